"""What the operators on device memory are measured on: the paged append, the
paged attention over shared prefixes, and the sampling of answer rows.

A state's K/V rows live in pages of a pool [pages, page, 2, kv_heads,
head_dim]; a group is a prefix (its own pages) and the branches that continue
from it, each a sequence with pages of its own. ``run`` computes a case in
plain torch operations, or with ``own`` set through grande_b200.ops.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -------------------------------------------------------------------

def _append(name, groups, prefix, branches, past, new, ragged, heads, kv_heads, head_dim,
            rope_dims, page, src, dtype, norm, v_norm):
    return {"name": name, "op": "append", "groups": groups, "prefix": prefix,
            "branches": branches, "past": past, "new": new, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rope_dims": rope_dims, "page": page,
            "src": src, "dtype": dtype, "norm": norm, "v_norm": v_norm}


def _attention(name, groups, prefix, branches, past, new, ragged, heads, kv_heads, head_dim,
               window, page, dtype):
    return {"name": name, "op": "attention", "groups": groups, "prefix": prefix,
            "branches": branches, "past": past, "new": new, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "page": page,
            "dtype": dtype}


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p, mixed, masked):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "mixed": mixed, "masked": masked}


def listed():
    return [
        # One answer token for each of 5 branches of a 90-token state, at the
        # 270M shape (4 query heads over one K/V head): a launch's latency.
        _append("append-token-270m", 1, 90, 5, 12, 1, False, 4, 1, 256, 256, 16, "f32", "f16",
                True, False),
        # 12 question branches of 24 tokens after a 2,000-token state, a
        # 512-dim global layer that rotates a quarter of each head and
        # normalises its values.
        _append("append-branches-hd512", 1, 2000, 12, 0, 24, False, 8, 2, 512, 128, 64, "f32",
                "f16", True, True),
        # A slice of 4 long prompts: 4,096 new tokens each, far positions.
        _append("append-prompt-bf16", 4, 0, 1, 28000, 4096, True, 16, 4, 128, 128, 32, "bf16",
                "bf16", True, False),
        # One answer token for each of 5 branches of a 90-token state.
        _attention("attend-token-270m", 1, 90, 5, 12, 1, True, 4, 1, 256, 0, 16, "f16"),
        # One answer token for each of 12 branches of a resident 2,000-token
        # state, a global layer and a sliding one.
        _attention("attend-token-e2b", 1, 2000, 12, 24, 1, True, 8, 2, 256, 0, 16, "f16"),
        _attention("attend-token-e2b-sliding", 1, 2000, 12, 24, 1, True, 8, 2, 256, 512, 16,
                   "f16"),
        # 64 resident states of 2,000 tokens with 20 branches each, one token
        # for every branch: the throughput of a full server.
        _attention("attend-token-64-states", 64, 2000, 20, 31, 1, True, 8, 2, 256, 0, 64, "f16"),
        # 12 question branches of 24 tokens against a 2,000-token state in a
        # 512-dim global layer.
        _attention("attend-branches-hd512", 1, 2000, 12, 0, 24, False, 8, 2, 512, 0, 64, "f16"),
        # 64 unrelated sequences of up to 8,192 tokens: no prefix to share.
        _attention("attend-token-ragged-bf16", 1, 0, 64, 8191, 1, True, 16, 4, 128, 0, 32,
                   "bf16"),
        # Answer tokens of 5 branches over the pruned vocabulary.
        _sample("sample-5-k64", 5, 25000, "f32", 1.0, 64, 0.95, 0.0, False, 0.0),
        # The whole distribution, every row with settings of its own.
        _sample("sample-64-mixed", 64, 56000, "bf16", 0.8, 200, 0.9, 0.02, True, 0.5),
        # A full server's rows over an unpruned vocabulary, cut by mass alone.
        _sample("sample-128-p90", 128, 262144, "f32", 1.0, 0, 0.9, 0.0, False, 0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "sample"])
    if op == "sample":
        vocab = _log_int(rng, 300, 262144)
        rows = _log_int(rng, 1, min(512, 128 * 262144 // vocab))
        c = _sample("", rows, vocab, rng.choice(["f32", "f16", "bf16"]),
                    rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.7]),
                    rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]),
                    rng.choice([1.0, 1.0, round(rng.uniform(0.05, 0.99), 3)]),
                    rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.5), 4)]),
                    rng.random() < 0.5, rng.choice([0.0, 0.5, 0.999]))
        del c["name"]
        return c
    head_dim = rng.choice([64, 128, 256, 256, 512])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    ragged = rng.random() < 0.7
    row = 4 * kv_heads * head_dim  # bytes of a cache row
    groups = _log_int(rng, 1, 64)
    branches = _log_int(rng, 1, 64)
    if op == "append":
        new = rng.choice([1, _log_int(rng, 1, 4096)])
        prefix = rng.choice([0, _log_int(rng, 1, 100000)])
        past = rng.choice([0, _log_int(rng, 1, 30000)])
        width = (heads + 2 * kv_heads) * head_dim
        while groups * branches * new * width > 12_000_000 and groups * branches * new > 1:
            groups, branches, new = (max(1, groups // 2), max(1, branches // 2),
                                     max(1, 2 * new // 3))
        while (groups * branches * (past + new)) * row > 200_000_000 and past:
            past //= 2
        dtype = rng.choice(["f16", "bf16"])
        c = _append("", groups, prefix, branches, past, new, ragged, heads, kv_heads, head_dim,
                    rng.choice([0, head_dim // 4, head_dim // 2, head_dim]), page,
                    rng.choice(["f32", dtype]), dtype, rng.random() < 0.7, rng.random() < 0.4)
    else:
        new = rng.choice([1, 1, _log_int(rng, 2, 200)])
        prefix = rng.choice([0, _log_int(rng, 1, 32000)])
        past = rng.choice([0, _log_int(rng, 1, 8000)])
        while groups > 1 and groups * prefix * row > 120_000_000:
            groups //= 2
        while groups * branches > 1 and groups * branches * (past + new) * row > 120_000_000:
            groups, branches = max(1, groups // 2), max(1, branches // 2)
        pairs = groups * branches * new * (prefix + past + new)
        while pairs * heads * head_dim > 4_000_000_000 and pairs > prefix + past + 1:
            groups, branches, new = (max(1, groups // 2), max(1, branches // 2),
                                     max(1, 2 * new // 3))
            pairs = groups * branches * new * (prefix + past + new)
        c = _attention("", groups, prefix, branches, past, new, ragged, heads, kv_heads, head_dim,
                       rng.choice([0, 0, 512, _log_int(rng, 1, 4000)]), page,
                       rng.choice(["f16", "bf16"]))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------

def _batch(case, g):
    """The page tables and lengths a serving loop keeps: host lists and the
    device tensors made from them. Pages are handed out in random order."""
    page, n_groups, n_br = case["page"], case["groups"], case["branches"]
    n_seq = n_groups * n_br
    # Ragged lengths belong to the case: every seed's outputs have one shape.
    gl = torch.Generator().manual_seed(n_seq + 64 * case["past"] + case["new"])
    past = [case["past"]] * n_seq
    if case["ragged"]:
        past = torch.randint(0, case["past"] + 1, (n_seq,), generator=gl).tolist()
    new = [case["new"]] * n_seq
    if case["ragged"] and case["new"] > 1:
        new = torch.randint(1, case["new"] + 1, (n_seq,), generator=gl).tolist()
    prefix = [case["prefix"]] * n_groups
    if case["ragged"] and n_groups > 1 and case["prefix"]:
        prefix = torch.randint(case["prefix"] // 2, case["prefix"] + 1, (n_groups,),
                               generator=gl).tolist()
    lens = [a + b for a, b in zip(past, new)]
    own_pages = [-(-n // page) for n in lens]
    pre_pages = [-(-n // page) for n in prefix]
    if case["op"] == "append":
        filled = [0] * n_groups  # the prefixes are not read: one page stands for all of theirs
    else:
        filled = pre_pages
    used = sum(own_pages) + sum(filled)
    total = used + 1
    order = torch.randperm(total, generator=g).tolist()
    width, pwidth = max(own_pages), max(max(pre_pages), 1)
    table = np.full((n_seq, width), order[-1], np.int32)
    ptable = np.full((n_groups, pwidth), order[-1], np.int32)
    at = 0
    for t, counts in ((ptable, filled), (table, own_pages)):
        for i, n in enumerate(counts):
            t[i, :n] = order[at:at + n]
            at += n
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    group_start = (np.arange(n_groups + 1) * n_br).astype(np.int32)
    dev = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in {
        "q_start": q_start, "lens": np.array(lens, np.int32), "pages": table,
        "group_start": group_start, "prefix_lens": np.array(prefix, np.int32),
        "prefix_pages": ptable}.items()}
    host = {"new": new, "lens": lens, "prefix": prefix, "table": table, "ptable": ptable,
            "tokens": int(q_start[-1]), "total": total}
    return host, dev


def _normal(shape, dtype, gd, scale=1.0):
    return (torch.randn(shape, generator=gd, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g, gd)
    host, dev = _batch(case, g)
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    st = {"case": case, "host": host, "dev": dev,
          "cache": _normal((host["total"], page, 2, kvh, hd), dt, gd)}
    if case["op"] == "append":
        st["qkv"] = _normal((host["tokens"], (heads + 2 * kvh) * hd), DTYPES[case["src"]], gd, 2.0)
        st["q_norm"] = st["k_norm"] = st["freq"] = None
        if case["norm"]:
            st["q_norm"] = _normal((hd,), torch.float32, gd, 0.1)
            st["k_norm"] = _normal((hd,), torch.float32, gd, 0.1)
        if case["rope_dims"]:
            # theta 1e6 over the whole head, the positions stretched by 8.
            d = np.arange(case["rope_dims"] // 2, dtype=np.float64)
            st["freq"] = torch.from_numpy(1e6 ** (-2.0 * d / hd) / 8.0).cuda()
        st["q_scale"] = hd ** -0.5
    else:
        st["q"] = _normal((host["tokens"], heads, hd), dt, gd)
        # Queries are scaled as they leave the append: scores of unit spread.
        st["scale"] = hd ** -0.5
    if own:
        from grande_b200 import ops
        st["batch"] = ops.PagedBatch(**dev)
    return st


def _prepare_sample(case, g, gd):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn((rows, vocab), generator=gd, device="cuda") * 2.5
    # A few likely tokens per row, as a trained model's rows have.
    hot = torch.randint(0, vocab, (rows, 8), generator=gd, device="cuda")
    x.scatter_add_(1, hot, torch.rand((rows, 8), generator=gd, device="cuda") * 10)
    if case["masked"]:
        # Tokens a constraint forbids.
        x[torch.rand((rows, vocab), generator=gd, device="cuda") < case["masked"]] = -math.inf
    f = torch.full
    st = {"case": case, "logits": x.to(DTYPES[case["dtype"]]),
          "u": torch.rand((rows,), generator=gd, device="cuda"),
          "temperature": f((rows,), case["temperature"], device="cuda"),
          "top_k": f((rows,), case["top_k"], dtype=torch.int32, device="cuda"),
          "top_p": f((rows,), case["top_p"], device="cuda"),
          "min_p": f((rows,), case["min_p"], device="cuda")}
    if case["mixed"]:
        # Requests with settings of their own: some of them greedy, some with
        # a filter off.
        pick = torch.randint(0, 4, (4, rows), generator=g).cuda()
        st["temperature"] = torch.where(pick[0] == 0, 0.0, st["temperature"])
        st["top_k"] = torch.where(pick[1] == 0, 0, st["top_k"] * pick[1]).to(torch.int32)
        st["top_p"] = torch.where(pick[2] == 0, 1.0, st["top_p"] ** pick[2])
        st["min_p"] = torch.where(pick[3] == 0, 0.0, (st["min_p"] * pick[3]).clamp(max=1))
    return st


# ---- one pass ----------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        from grande_b200 import ops
        if case["op"] == "append":
            q = ops.paged_append(state["qkv"], state["cache"], state["batch"],
                                 heads=case["heads"], q_norm=state["q_norm"],
                                 k_norm=state["k_norm"], norm_offset=1.0, eps=1e-6,
                                 v_norm=case["v_norm"], inv_freq=state["freq"],
                                 q_scale=state["q_scale"])
            return {"q": q, "cache": state["cache"]}
        if case["op"] == "attention":
            return {"out": ops.paged_attention(state["q"], state["cache"], state["batch"],
                                               scale=state["scale"], window=case["window"])}
        tokens, probs = ops.sample(state["logits"], state["u"],
                                   temperature=state["temperature"], top_k=state["top_k"],
                                   top_p=state["top_p"], min_p=state["min_p"])
        return {"tokens": tokens, "probs": probs}
    return {"append": _plain_append, "attention": _plain_attention,
            "sample": _plain_sample}[case["op"]](state)


def _token_index(dev):
    """Per token: its sequence, its index among the sequence's own tokens, its
    position."""
    q_start, lens = dev["q_start"].long(), dev["lens"].long()
    n = q_start[1:] - q_start[:-1]
    n_seq = n.numel()
    seq = torch.repeat_interleave(torch.arange(n_seq, device=n.device), n)
    idx = torch.arange(seq.numel(), device=n.device) - q_start[seq] + lens[seq] - n[seq]
    group = torch.searchsorted(dev["group_start"].long(), seq, right=True) - 1
    return seq, idx, idx + dev["prefix_lens"].long()[group], group


def _plain_append(st):
    case, dev, cache = st["case"], st["dev"], st["cache"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = st["qkv"].float().view(-1, heads + 2 * kvh, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]

    def rms(y):
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)

    if st["q_norm"] is not None:
        q, k = rms(q) * (1.0 + st["q_norm"]), rms(k) * (1.0 + st["k_norm"])
    if case["v_norm"]:
        v = rms(v)
    seq, idx, pos, _ = _token_index(dev)
    if st["freq"] is not None:
        a = pos.double()[:, None] * st["freq"]
        cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
        n = st["freq"].numel()

        def rot(y):
            lo, hi = y[..., :n], y[..., hd // 2:hd // 2 + n]
            out = y.clone()
            out[..., :n] = lo * cos - hi * sin
            out[..., hd // 2:hd // 2 + n] = hi * cos + lo * sin
            return out

        q, k = rot(q), rot(k)
    pg = dev["pages"].long()[seq, idx // page]
    cache[pg, idx % page] = torch.stack([k, v], 1).to(cache.dtype)
    return {"q": (q * st["q_scale"]).to(cache.dtype), "cache": cache}


def _plain_attention(st):
    case, dev, cache, host = st["case"], st["dev"], st["cache"], st["host"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    window, q = case["window"], st["q"]
    hpg = heads // kvh
    out = torch.empty_like(q)
    t0 = 0
    for grp in range(case["groups"]):
        lo, hi = grp * case["branches"], (grp + 1) * case["branches"]
        new, lens = host["new"][lo:hi], host["lens"][lo:hi]
        pre, t1 = host["prefix"][grp], t0 + sum(new)
        # The group's queries padded to [branches, new, kv_heads, hpg, hd].
        n = torch.tensor(new, device=q.device)
        live = torch.arange(max(new), device=q.device) < n[:, None]
        qs = q.new_zeros((hi - lo, max(new), heads, hd), dtype=torch.float32)
        qs[live] = q[t0:t1].float()
        qs = qs.view(hi - lo, max(new), kvh, hpg, hd)
        own_idx = (torch.tensor(lens, device=q.device) - n)[:, None] + torch.arange(
            max(new), device=q.device)
        most = max(lens)
        rows = cache[dev["pages"][lo:hi, :-(-most // page)].long()].flatten(1, 2)[:, :most].float()
        keys, vals = rows[:, :, 0], rows[:, :, 1]
        j = torch.arange(most, device=q.device)
        seen = j <= own_idx[..., None]
        if window:
            seen &= j > own_idx[..., None] - window
        s = torch.einsum("bqghd,bkgd->bqghk", qs, keys) * st["scale"]
        s = s.masked_fill(~seen[:, :, None, None], -math.inf)
        vals = vals.masked_fill((j >= torch.tensor(lens, device=q.device)[:, None])[..., None, None],
                                0)
        if pre:
            pt = dev["prefix_pages"][grp, :-(-pre // page)].long()
            prow = cache[pt].flatten(0, 1)[:pre].float()
            ps = torch.einsum("bqghd,kgd->bqghk", qs, prow[:, 0]) * st["scale"]
            if window:
                jp = torch.arange(pre, device=q.device)
                ps = ps.masked_fill(~(jp > own_idx[..., None] + pre - window)[:, :, None, None],
                                    -math.inf)
            s = torch.cat([ps, s], -1)
        s = s - s.amax(-1, keepdim=True)
        p = s.exp()
        p = p / p.sum(-1, keepdim=True)
        o = torch.einsum("bqghk,bkgd->bqghd", p[..., pre:], vals)
        if pre:
            o = o + torch.einsum("bqghk,kgd->bqghd", p[..., :pre], prow[:, 1])
        out[t0:t1] = o.flatten(2, 3)[live].to(out.dtype)
        t0 = t1
    return {"out": out}


def _plain_sample(st):
    x = st["logits"].double()
    rows, vocab = x.shape
    greedy = st["temperature"] <= 0
    temp = torch.where(greedy, 1.0, st["temperature"].double())[:, None]
    k = torch.where(greedy, 1, torch.where(st["top_k"] > 0, st["top_k"], vocab)).long()[:, None]
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    dead = xs[:, 0] == -math.inf  # no token is left: -1, of probability 0
    w = ((xs - xs[:, :1].clamp(min=-1e300)) / temp).exp()
    w = torch.where(torch.arange(vocab, device=x.device) < k, w, 0.0)
    cum = w.cumsum(1)
    before = cum.roll(1, 1)
    before[:, 0] = 0
    target = st["top_p"].double()[:, None] * cum[:, -1:]
    w = torch.where((before < target) | (st["top_p"][:, None] >= 1), w, 0.0)
    w = torch.where(w >= st["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = w.cumsum(1)
    total = cum[:, -1:]
    tok = (cum <= st["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    prob = (w.gather(1, tok) / total)[:, 0]
    return {"tokens": torch.where(dead, -1, tok[:, 0]).to(torch.int32),
            "probs": torch.where(dead, 0.0, prob).float()}


# ---- the definition in 64 bits ------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention,
            "sample": _exact_sample}[case["op"]](st)


def _exact_append(st):
    case, host = st["case"], st["host"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = st["qkv"].double().reshape(host["tokens"], heads + 2 * kvh, hd)
    norm = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
    if st["q_norm"] is not None:
        w = torch.cat([st["q_norm"].double().expand(heads, hd),
                       st["k_norm"].double().expand(kvh, hd)]) + 1.0
        x = torch.cat([norm[:, :heads + kvh] * w, x[:, heads + kvh:]], 1)
    if case["v_norm"]:
        x = torch.cat([x[:, :heads + kvh], norm[:, heads + kvh:]], 1)
    slots, pos = [], []
    s = 0
    for grp in range(case["groups"]):
        for _ in range(case["branches"]):
            i = np.arange(host["lens"][s] - host["new"][s], host["lens"][s])
            slots.append(host["table"][s][i // page].astype(np.int64) * page + i % page)
            pos.append(i + host["prefix"][grp])
            s += 1
    slots = torch.from_numpy(np.concatenate(slots)).cuda()
    if st["freq"] is not None:
        n = st["freq"].numel()
        a = torch.from_numpy(np.concatenate(pos).astype(np.float64)).cuda()[:, None, None] * st["freq"]
        turn = torch.polar(torch.ones_like(a), a)
        z = torch.complex(x[:, :heads + kvh, :n], x[:, :heads + kvh, hd // 2:hd // 2 + n]) * turn
        x[:, :heads + kvh, :n], x[:, :heads + kvh, hd // 2:hd // 2 + n] = z.real, z.imag
    flat = st["cache"].double().reshape(-1, 2 * kvh * hd)
    flat[slots] = x[:, heads:].reshape(-1, 2 * kvh * hd)
    return {"q": x[:, :heads] * st["q_scale"], "cache": flat.view(st["cache"].shape)}


def _exact_attention(st):
    case, host = st["case"], st["host"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    cache = st["cache"].reshape(-1, 2, kvh, hd)
    pairs = sum(n * (length + host["prefix"][s // case["branches"]])
                for s, (n, length) in enumerate(zip(host["new"], host["lens"])))
    if pairs * heads > 600_000_000:
        return None
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")

    def rows(table, n):
        j = np.arange(n)
        at = table[j // page].astype(np.int64) * page + j % page
        return cache[torch.from_numpy(at).cuda()].double()

    t = 0
    for s, (n, length) in enumerate(zip(host["new"], host["lens"])):
        pre = host["prefix"][s // case["branches"]]
        if s % case["branches"] == 0:
            head = rows(host["ptable"][s // case["branches"]], pre)
        kv = torch.cat([head, rows(host["table"][s], length)])
        at = torch.arange(pre + length - n, pre + length, device="cuda")
        key = torch.arange(pre + length, device="cuda")
        hide = key[None] > at[:, None]
        if case["window"]:
            hide |= at[:, None] - key[None] >= case["window"]
        for h in range(kvh):
            q = st["q"][t:t + n, h * (heads // kvh):(h + 1) * (heads // kvh)].double()
            z = torch.matmul(q, kv[:, 0, h].T) * st["scale"]
            z = torch.softmax(z.masked_fill(hide[:, None], -math.inf), -1)
            out[t:t + n, h * (heads // kvh):(h + 1) * (heads // kvh)] = torch.matmul(z, kv[:, 1, h])
        t += n
    return {"out": out}


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    par = {k: st[k].cpu().numpy() for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    toks, probs = [], []
    for r in range(x.shape[0]):
        row, temp, k = x[r], float(par["temperature"][r]), int(par["top_k"][r])
        if row.max() == -math.inf:
            toks.append(-1)
            probs.append(0.0)
            continue
        if temp <= 0:
            toks.append(int(row.argmax()))
            probs.append(1.0)
            continue
        rank = np.argsort(-row, kind="stable")
        if k > 0:
            rank = rank[:k]
        mass = np.exp((row[rank] - row[rank[0]]) / temp)
        if par["top_p"][r] < 1:
            goal = float(par["top_p"][r]) * mass.sum()
            n = int(np.searchsorted(np.cumsum(mass), goal, side="left")) + 1
            rank, mass = rank[:n], mass[:n]
        good = mass >= float(par["min_p"][r])
        rank, mass = rank[good], mass[good]
        by_id = np.argsort(rank, kind="stable")
        rank, mass = rank[by_id], mass[by_id]
        run_sum = np.cumsum(mass)
        at = int(np.searchsorted(run_sum, float(par["u"][r]) * run_sum[-1], side="right"))
        at = min(at, len(rank) - 1)
        toks.append(int(rank[at]))
        probs.append(float(mass[at] / run_sum[-1]))
    return {"tokens": torch.tensor(toks, dtype=torch.int32),
            "probs": torch.tensor(probs, dtype=torch.float64)}


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    """Each input read once and each output written once; ragged lengths at
    their mean."""
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * 28, "flops": 2 * n}
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    seqs = case["groups"] * case["branches"]
    past = case["past"] / 2 if case["ragged"] else case["past"]
    new = (1 + case["new"]) / 2 if case["ragged"] and case["new"] > 1 else case["new"]
    pre = case["prefix"] * (0.75 if case["ragged"] and case["groups"] > 1 else 1.0)
    tokens = seqs * new
    if case["op"] == "append":
        return {"bytes": int(tokens * hd * ((heads + 2 * kvh) * (SIZE[case["src"]] + 2))),
                "flops": int(tokens * (heads + 2 * kvh) * hd * 8)}
    if case["window"]:
        seen = min(case["window"], pre + past + new / 2)
        own_rows = min(past + new, case["window"] + new)
        pre_rows = max(0, min(pre, case["window"] + new - past))
    else:
        seen, own_rows, pre_rows = pre + past + new / 2, past + new, pre
    kv = (case["groups"] * pre_rows + seqs * own_rows) * 2 * kvh * hd * 2
    return {"bytes": int(kv + 2 * tokens * heads * hd * 2),
            "flops": int(4 * tokens * heads * hd * seen)}
