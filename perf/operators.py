"""The attention, cache and verification operators: what is measured, and their plain forms.

A case is one pass through one operator as a serving loop calls it. `run` computes it with
elementary torch operations, or through the library's own entry points where `own` is true.

kind "prompt"  causal attention over packed whole prompts (sllm_cuda_attn_prompt)
kind "prefix"  decode attention of sequences that share a prefix (sllm_cuda_attn_prefix)
kind "fork"    sequences forked, then pages reserved for their next tokens (sllm_cuda_kv_fork, _reserve)
kind "compact" a fragmented cache compacted (sllm_cuda_kv_compact)
kind "append"  RoPE, conversion and page store of new tokens (sllm_cuda_kv_append)
kind "verify"  drafted tokens verified against the target's probabilities (sllm_cuda_spec_verify)
"""
import importlib
import math

import numpy as np
import torch

own = False

D = 128                       # the head dimension of every model the library runs
SCALE = 1.0 / math.sqrt(D)


def listed():
    return [
        # one user's short prompt through the 2B-4T heads: the smallest call, latency
        {"name": "prompt_short_f16", "kind": "prompt", "f16": True, "H": 20, "Hkv": 5, "lens": "17"},
        # a prefill batch through the 64/8 heads of the 80-layer model: long, short, empty and odd prompts packed
        {"name": "prompt_packed_f16", "kind": "prompt", "f16": True, "H": 64, "Hkv": 8,
         "lens": "8192,1,300,1021,0,2048,513,64"},
        # prompts in the library's default f32, 2B-4T heads
        {"name": "prompt_f32", "kind": "prompt", "f16": False, "H": 20, "Hkv": 5, "lens": "320,1,777,256"},
        # two conversations over one system prompt, f32 cache, small pages
        {"name": "prefix_small_f32", "kind": "prefix", "f16": False, "H": 20, "Hkv": 5, "n": 2, "nq": 1,
         "prefix": 256, "own": 64, "page": 16, "layers": 2},
        # a batch of 16 over a 4k system prompt, one decode step
        {"name": "prefix_batch_f16", "kind": "prefix", "f16": True, "H": 20, "Hkv": 5, "n": 16, "nq": 1,
         "prefix": 4096, "own": 300, "page": 16, "layers": 1},
        # 64 sequences over a 32k document, each with three drafted tokens to score
        {"name": "prefix_draft_f16", "kind": "prefix", "f16": True, "H": 64, "Hkv": 8, "n": 64, "nq": 4,
         "prefix": 32768, "own": 1000, "page": 64, "layers": 1},
        # four samples of one prompt: fork, then the first write to the shared last page
        {"name": "pages_fork", "kind": "fork", "f16": True, "Hkv": 5, "page": 16, "layers": 30, "parents": 1,
         "children": 4, "len": 301, "new": 1, "spare": 40},
        # a cache whose finished conversations left holes, compacted
        {"name": "pages_compact", "kind": "compact", "f16": True, "Hkv": 5, "page": 16, "layers": 30, "slots": 48,
         "len": 200, "pages": 1024},
        # one decode step's new tokens of a batch of 16
        {"name": "append_step_f16", "kind": "append", "f16": True, "H": 20, "Hkv": 5, "T": 16, "slots": 16,
         "page": 16, "layers": 2},
        # a prefill's tokens into an f32 cache
        {"name": "append_prompt_f32", "kind": "append", "f16": False, "H": 64, "Hkv": 8, "T": 4099, "slots": 5,
         "page": 64, "layers": 1},
        # one sequence's four drafted tokens over the 128256-word vocabulary
        {"name": "verify_one", "kind": "verify", "n": 1, "k": 4, "V": 128256, "point": False},
        # a batch's seven drafted tokens, lengths of drafts differing
        {"name": "verify_batch", "kind": "verify", "n": 64, "k": 7, "V": 128256, "point": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice([(20, 5), (64, 8), (8, 1), (4, 4), (6, 2), (14, 2)])
    kind = rng.choice(["prompt", "prefix", "fork", "compact", "append", "verify"])
    f16 = rng.random() < 0.7
    page = rng.choice([16, 32, 64, 128])
    if kind == "prompt":
        lens = [_log(rng, 1, 2500 if f16 else 900) for _ in range(rng.randint(1, 9))]
        if rng.random() < 0.3:
            lens.insert(rng.randrange(len(lens) + 1), 0)
        return {"kind": kind, "f16": f16, "H": heads[0], "Hkv": heads[1], "lens": ",".join(map(str, lens))}
    if kind == "prefix":
        n = _log(rng, 1, 64 if f16 else 12)
        nq = rng.choice([1, 1, 2, 3, 4, 5, 8])
        return {"kind": kind, "f16": f16, "H": heads[0], "Hkv": heads[1], "n": n, "nq": nq,
                "prefix": page * rng.randint(0, 8) if rng.random() < 0.3 else page * (_log(rng, page, 16000) // page),
                "own": _log(rng, nq, 1000), "page": page, "layers": rng.randint(1, 2)}
    if kind == "fork":
        return {"kind": kind, "f16": f16, "Hkv": heads[1], "page": page, "layers": rng.randint(1, 8),
                "parents": rng.randint(1, 6), "children": rng.randint(1, 9), "len": _log(rng, 1, 600),
                "new": rng.choice([0, 1, 1, 5, 70]), "spare": 3000 // page}
    if kind == "compact":
        slots = rng.randint(1, 60)
        length = _log(rng, 1, 400)
        return {"kind": kind, "f16": f16, "Hkv": heads[1], "page": page, "layers": rng.randint(1, 4),
                "slots": slots, "len": length, "pages": 2 * slots * (length // page + 1) + rng.randint(1, 50)}
    if kind == "append":
        return {"kind": kind, "f16": f16, "H": heads[0], "Hkv": heads[1], "T": _log(rng, 1, 4000),
                "slots": rng.randint(1, 16), "page": page, "layers": rng.randint(1, 3)}
    return {"kind": "verify", "n": _log(rng, 1, 64), "k": rng.randint(1, 8), "V": _log(rng, 2, 128256),
            "point": rng.random() < 0.3}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dt(case):
    return torch.float16 if case["f16"] else torch.float32


def _normal(g, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _own_lens(case, seed):
    """Each sequence's own tokens after the prefix: at least the query tokens, up to `own`."""
    r = np.random.default_rng(seed)
    lo = min(case["nq"], case["own"])
    return [int(x) for x in r.integers(lo, case["own"] + 1, case["n"])]


def _draft_lens(case, seed):
    r = np.random.default_rng(seed + 1)
    return [int(x) for x in r.integers(min(1, case["k"]), case["k"] + 1, case["n"])] if case["n"] > 1 else [case["k"]]


def _pkg():
    return importlib.import_module("saphira-llm_b200")


def _handle(case, st):
    """The library's view of a paged cache and its scratch, kept as a server keeps them."""
    if own:
        st["pages"] = _pkg().KvPages(st["k"], st["v"], st["refs"], st["tables"], st["lens"])
        st["work"] = torch.empty(st["pages"].work_bytes(), dtype=torch.uint8, device="cuda")
    return st


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "prompt":
        lens = [int(x) for x in case["lens"].split(",")]
        T, H, Hkv, dt = sum(lens), case["H"], case["Hkv"], _dt(case)
        # queries and keys as the projections leave them, a little peaked; one tensor as a fused Q/K/V product gives
        qkv = _normal(g, (T, H + 2 * Hkv, D), dt)
        qkv[:, :H] *= 1.5
        cu = np.concatenate([[0], np.cumsum(lens)])
        return {"case": case, "lens": lens, "cu": _i32(cu.tolist()), "q": qkv[:, :H], "k": qkv[:, H:H + Hkv],
                "v": qkv[:, H + Hkv:], "out": torch.empty((T, H, D), dtype=dt, device="cuda")}
    if kind == "prefix":
        dt, page, n = _dt(case), case["page"], case["n"]
        owns = _own_lens(case, seed)
        npre = case["prefix"] // page
        need = npre + sum((o + page - 1) // page for o in owns)
        n_pages = need + 7
        r = np.random.default_rng(seed + 2)
        ids = r.permutation(n_pages)[:need]                  # a used cache hands out pages in no order
        width = npre + (max(owns) + page - 1) // page + 1
        tab = np.full((n + 2, width), -1, np.int64)
        refs = np.zeros(n_pages, np.int64)
        at = npre
        slots = r.permutation(n + 2)[:n]
        lens = np.zeros(n + 2, np.int64)
        for s, o in zip(slots, owns):
            m = (o + page - 1) // page
            tab[s, :npre] = ids[:npre]
            tab[s, npre:npre + m] = ids[at:at + m]
            at += m
            lens[s] = case["prefix"] + o
            refs[ids[:npre]] += 1
            refs[tab[s, npre:npre + m]] += 1
        shape = (n_pages, case["layers"], case["Hkv"], page, D)
        st = {"case": case, "owns": owns, "layer": case["layers"] - 1, "k": _normal(g, shape, dt),
              "v": _normal(g, shape, dt), "refs": _i32(refs.tolist()), "tables": _i32(tab.tolist()),
              "lens": _i32(lens.tolist()), "slots": _i32(slots.tolist()),
              "q": _normal(g, (n, case["nq"], case["H"], D), dt, 1.5),
              "out": torch.empty((n, case["nq"], case["H"], D), dtype=dt, device="cuda"),
              "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
        _handle(case, st)
        if own:
            st["scratch"] = torch.empty(st["pages"].attn_prefix_work_bytes(n, case["nq"], case["H"], case["prefix"]),
                                        dtype=torch.uint8, device="cuda")
        return st
    if kind == "fork":
        dt, page = _dt(case), case["page"]
        r = np.random.default_rng(seed)
        P, Cn = case["parents"], case["children"]
        plens = [max(1, case["len"] - int(r.integers(0, max(1, min(case["len"], 2 * page))))) for _ in range(P)]
        plens[0] = case["len"]
        used = [(x + page - 1) // page for x in plens]
        per = (case["len"] + case["new"] + page - 1) // page + 1
        n_slots = P * (1 + Cn)
        n_pages = P * max(used) + n_slots * (case["new"] // page + 2) + case["spare"]
        ids = r.permutation(n_pages)
        tab = np.full((n_slots, per), -1, np.int64)
        refs = np.zeros(n_pages, np.int64)
        lens = np.zeros(n_slots, np.int64)
        at = 0
        for p in range(P):
            tab[p, :used[p]] = ids[at:at + used[p]]
            refs[tab[p, :used[p]]] = 1
            lens[p] = plens[p]
            at += used[p]
        src = [p for p in range(P) for _ in range(Cn)]
        dst = list(range(P, n_slots))
        shape = (n_pages, case["layers"], case["Hkv"], page, D)
        st = {"case": case, "k": _normal(g, shape, dt), "v": _normal(g, shape, dt), "refs": _i32(refs.tolist()),
              "tables": _i32(tab.tolist()), "lens": _i32(lens.tolist()), "src": _i32(src), "dst": _i32(dst),
              "slots": _i32(list(range(n_slots))), "new": _i32([case["new"]] * n_slots),
              "plens": plens, "status": torch.zeros(2, dtype=torch.int32, device="cuda")}
        st["saved"] = [st[x].clone() for x in ("refs", "tables", "lens")]
        return _handle(case, st)
    if kind == "compact":
        dt, page, S = _dt(case), case["page"], case["slots"]
        r = np.random.default_rng(seed)
        lens = r.integers(0, case["len"] + 1, S)
        used = (lens + page - 1) // page
        ids = r.permutation(case["pages"])
        width = (case["len"] + page - 1) // page + 1
        tab = np.full((S, width), -1, np.int64)
        refs = np.zeros(case["pages"], np.int64)
        at = 0
        for s in range(S):
            share = min(int(used[s]), int(used[s - 1])) // 2 if s % 3 == 2 else 0    # some were forked
            full = min(share, int(lens[s - 1]) // page)
            tab[s, :full] = tab[s - 1, :full]
            tab[s, full:used[s]] = ids[at:at + used[s] - full]
            at += used[s] - full
            np.add.at(refs, tab[s, :used[s]], 1)
        shape = (case["pages"], case["layers"], case["Hkv"], page, D)
        st = {"case": case, "k": _normal(g, shape, dt), "v": _normal(g, shape, dt), "refs": _i32(refs.tolist()),
              "tables": _i32(tab.tolist()), "lens": _i32(lens.tolist()),
              "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
        st["saved"] = [st[x].clone() for x in ("refs", "tables", "lens")]
        return _handle(case, st)
    if kind == "append":
        dt, page, H, Hkv, T, S = _dt(case), case["page"], case["H"], case["Hkv"], case["T"], case["slots"]
        r = np.random.default_rng(seed)
        cnt = np.bincount(np.sort(r.integers(0, S, T)), minlength=S)
        past = r.integers(0, 2 * page + 1, S)
        lens = cnt + past
        used = (lens + page - 1) // page
        n_pages = (T + S * 2 * page) // page + S + 3
        ids = r.permutation(n_pages)
        tab = np.full((S, int(used.max()) + 1), -1, np.int64)
        at = 0
        refs = np.zeros(n_pages, np.int64)
        for s in range(S):
            tab[s, :used[s]] = ids[at:at + used[s]]
            refs[tab[s, :used[s]]] = 1
            at += used[s]
        slot = np.repeat(np.arange(S), cnt)
        pos = np.concatenate([past[s] + np.arange(cnt[s]) for s in range(S)])
        shape = (n_pages, case["layers"], Hkv, page, D)
        n_ctx = int(lens.max())
        ang = np.arange(n_ctx)[:, None] * (500000.0 ** (-2.0 * np.arange(D // 2) / D))[None]
        qkv = _normal(g, (T, H + 2 * Hkv, D), torch.float32)
        st = {"case": case, "layer": case["layers"] - 1, "k": torch.zeros(shape, dtype=dt, device="cuda"),
              "v": torch.zeros(shape, dtype=dt, device="cuda"), "refs": _i32(refs.tolist()),
              "tables": _i32(tab.tolist()), "lens": _i32(lens.tolist()), "slot": _i32(slot.tolist()),
              "pos": _i32(pos.tolist()), "cos": torch.tensor(np.cos(ang), dtype=torch.float32, device="cuda"),
              "sin": torch.tensor(np.sin(ang), dtype=torch.float32, device="cuda"), "qi": qkv[:, :H],
              "ki": qkv[:, H:H + Hkv], "vi": qkv[:, H + Hkv:], "qo": torch.empty((T, H, D), dtype=dt, device="cuda"),
              "ko": torch.empty((T, Hkv, D), dtype=dt, device="cuda"),
              "vo": torch.empty((T, Hkv, D), dtype=dt, device="cuda"),
              "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
        return _handle(case, st)
    # verify: a target and a draft that mostly agree, as a trained pair does
    n, k, V = case["n"], case["k"], case["V"]
    logits = torch.randn((n, k + 1, V), generator=g, device="cuda") * 3.0
    p = torch.softmax(logits, -1)
    noise = torch.randn((n, k, V), generator=g, device="cuda") * 0.7
    q = torch.softmax(logits[:, :k] + noise, -1)
    del logits, noise
    draft = torch.multinomial(q.reshape(n * k, V), 1, generator=g).reshape(n, k).to(torch.int32)
    return {"case": case, "p": p, "q": None if case["point"] else q, "draft": draft,
            "nd": _i32(_draft_lens(case, seed)), "ua": torch.rand((n, k), generator=g, device="cuda"),
            "us": torch.rand((n,), generator=g, device="cuda"),
            "tokens": torch.empty((n, k + 1), dtype=torch.int32, device="cuda"),
            "count": torch.empty((n,), dtype=torch.int32, device="cuda")}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_prompt(st):
    case, out = st["case"], st["out"]
    H, Hkv = case["H"], case["Hkv"]
    G = H // Hkv
    at = 0
    for L in st["lens"]:
        if L == 0:
            continue
        q = st["q"][at:at + L].float().view(L, Hkv, G, D).permute(1, 2, 0, 3)        # [Hkv, G, L, D]
        k = st["k"][at:at + L].float().permute(1, 2, 0)                              # [Hkv, D, L]
        v = st["v"][at:at + L].float().permute(1, 0, 2)                              # [Hkv, L, D]
        step = max(1, min(L, (1 << 28) // (H * L)))
        for a in range(0, L, step):
            b = min(L, a + step)
            s = torch.matmul(q[:, :, a:b], k[:, None, :, :b]) * SCALE                # [Hkv, G, b - a, b]
            i = torch.arange(a, b, device="cuda")[:, None]
            s = s.masked_fill(torch.arange(b, device="cuda")[None] > i, float("-inf"))
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(e, v[:, None, :b]) / e.sum(-1, keepdim=True)
            out[at + a:at + b] = o.permute(2, 0, 1, 3).reshape(b - a, H, D).to(out.dtype)
        at += L
    return out


def _plain_prefix(st):
    case, out = st["case"], st["out"]
    H, Hkv, page, n, nq, P = case["H"], case["Hkv"], case["page"], case["n"], case["nq"], case["prefix"]
    G = H // Hkv
    slots = st["slots"].long()
    tab = st["tables"][slots].long()
    lens = st["lens"][slots].long()
    npre, m = P // page, (max(st["owns"]) + page - 1) // page
    layer = st["layer"]
    own_ids = tab[:, npre:npre + m].clamp(min=0)                                     # [n, m]
    j = torch.arange(m * page, device="cuda")
    # query t of a sequence sees its first len - nq + 1 + t tokens
    limit = (lens[:, None] - nq + 1 + torch.arange(nq, device="cuda")[None]) - P     # [n, nq]
    for h in range(Hkv):
        q = st["q"][:, :, h * G:(h + 1) * G].float()                                 # [n, nq, G, D]
        ko = st["k"][:, layer, h][own_ids].float().reshape(n, m * page, D)
        vo = st["v"][:, layer, h][own_ids].float().reshape(n, m * page, D)
        so = torch.matmul(q.reshape(n, nq * G, D), ko.transpose(1, 2)).view(n, nq, G, m * page) * SCALE
        dead = (j[None, None] >= limit[:, :, None])[:, :, None]
        so = so.masked_fill(dead, float("-inf"))
        mx = so.amax(-1, keepdim=True)
        if npre:
            kp = st["k"][:, layer, h][tab[0, :npre]].float().reshape(P, D)
            vp = st["v"][:, layer, h][tab[0, :npre]].float().reshape(P, D)
            sp = torch.matmul(q.reshape(n * nq * G, D), kp.t()).view(n, nq, G, P) * SCALE
            mx = torch.maximum(mx, sp.amax(-1, keepdim=True))
        mx = torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)
        e = torch.exp(so - mx)
        den = e.sum(-1, keepdim=True)
        num = torch.matmul(e.view(n, nq * G, m * page), vo).view(n, nq, G, D)
        if npre:
            ep = torch.exp(sp - mx)
            den = den + ep.sum(-1, keepdim=True)
            num = num + torch.matmul(ep.view(n * nq * G, P), vp).view(n, nq, G, D)
        out[:, :, h * G:(h + 1) * G] = torch.where(den > 0, num / den, torch.zeros_like(num)).to(out.dtype)
    st["status"].zero_()
    return out


def _restore(st):
    for name, t in zip(("refs", "tables", "lens"), st["saved"]):
        st[name].copy_(t)


def _plain_fork(st):
    case = st["case"]
    page = case["page"]
    refs, tab, lens = st["refs"], st["tables"], st["lens"]
    width = tab.shape[1]
    col = torch.arange(width, device="cuda")[None]
    src, dst = st["src"].long(), st["dst"].long()
    # fork: what dst held is given back, then dst shares src's pages (all of them, the last one too)
    rows, rlen = tab[src], lens[src]
    live = col < ((rlen + page - 1) // page)[:, None]
    old, olen = tab[dst], lens[dst]
    olive = col < ((olen + page - 1) // page)[:, None]
    refs.index_add_(0, torch.where(live, rows, 0).reshape(-1).long(), live.reshape(-1).int())
    refs.index_add_(0, torch.where(olive, old, 0).reshape(-1).long(), -olive.reshape(-1).int())
    tab[dst] = torch.where(live, rows, old)
    lens[dst] = rlen
    # reserve: slots in order, each a copy of a shared last page if it will write there, then its new pages
    slots, new = st["slots"].long(), st["new"]
    n = slots.shape[0]
    cur = lens[slots]
    last = tab[slots, (cur // page).long().clamp(max=width - 1)]
    part = (cur % page != 0) & (new > 0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    rank = torch.tril(same, -1).sum(1)
    cow = part & (refs[last.long().clamp(min=0)] - rank > 1)
    fresh = (cur + new + page - 1) // page - (cur + page - 1) // page
    need = cow.int() + fresh
    first = torch.cumsum(need, 0) - need
    free = torch.sort((refs != 0).to(torch.int32), stable=True).indices.to(torch.int32)     # free pages, lowest first
    got = torch.where(cow, free[first.long().clamp(max=free.shape[0] - 1)], last)
    refs.index_add_(0, torch.where(cow, last, 0).long(), -cow.int())
    refs.index_add_(0, torch.where(cow, got, 0).long(), cow.int())
    rr = torch.arange(page, device="cuda")
    keep = cow[:, None] & (rr[None] < (cur % page)[:, None])                                # rows that are copied
    a, b = last.long().clamp(min=0), got.long().clamp(min=0)
    for pool in (st["k"], st["v"]):
        i = torch.nonzero(cow).squeeze(1)
        pool[b[i]] = torch.where(keep[i][:, None, None, :, None], pool[a[i]], pool[b[i]])
    at = (cur // page).long().clamp(max=width - 1)
    tab[slots, at] = torch.where(part, got, tab[slots, at])
    for x in range(case["new"] // page + 1):
        take = x < fresh
        ids = free[(first + cow.int() + x).long().clamp(max=free.shape[0] - 1)]
        where = ((cur + page - 1) // page + x).long().clamp(max=width - 1)
        tab[slots, where] = torch.where(take, ids, tab[slots, where])
        refs.index_add_(0, torch.where(take, ids, 0).long(), take.int())
    lens[slots] = cur + new
    st["status"].zero_()


def _plain_compact(st):
    refs, tab, lens, page = st["refs"], st["tables"], st["lens"], st["case"]["page"]
    live = refs > 0
    n_live = live.sum()
    idx = torch.arange(refs.shape[0], device="cuda")
    src = torch.nonzero(live & (idx >= n_live)).squeeze(1)
    dst = torch.nonzero(~live & (idx < n_live)).squeeze(1)
    st["k"][dst] = st["k"][src]
    st["v"][dst] = st["v"][src]
    remap = idx.clone()
    remap[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    used = torch.arange(tab.shape[1], device="cuda")[None] < ((lens + page - 1) // page)[:, None]
    tab.copy_(torch.where(used, remap[tab.long().clamp(min=0)].to(torch.int32), tab))
    st["status"].zero_()


def _plain_append(st):
    page = st["case"]["page"]
    dt = st["k"].dtype
    pos, slot = st["pos"].long(), st["slot"].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def rope(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1).to(dt)

    st["qo"].copy_(rope(st["qi"]))
    st["ko"].copy_(rope(st["ki"]))
    st["vo"].copy_(st["vi"].to(dt))
    ids = st["tables"][slot, pos // page].long()
    st["k"][ids, st["layer"], :, pos % page] = st["ko"]
    st["v"][ids, st["layer"], :, pos % page] = st["vo"]
    st["status"].zero_()


def _plain_verify(st):
    p, q, draft = st["p"], st["q"], st["draft"].long()
    n, k, V = draft.shape[0], draft.shape[1], p.shape[2]
    t = torch.arange(k, device="cuda")[None]
    px = torch.gather(p[:, :k], 2, draft[..., None]).squeeze(2).double()
    qx = torch.ones_like(px) if q is None else torch.gather(q, 2, draft[..., None]).squeeze(2).double()
    ok = (st["ua"].double() * qx < px) & (t < st["nd"][:, None])
    r = torch.cumprod(ok.int(), 1).sum(1)                                    # accepted tokens
    i = torch.arange(n, device="cuda")
    row = p[i, r].double()
    refused = r < st["nd"]
    rc = r.clamp(max=k - 1)
    if q is None:
        sub = torch.zeros_like(row)
        sub[i, draft[i, rc]] = row[i, draft[i, rc]]
    else:
        sub = q[i, rc].double()
    res = torch.where(refused[:, None], (row - sub).clamp(min=0), row)
    has = res.sum(1) > 0
    res = torch.where(has[:, None], res, row)
    cum = torch.cumsum(res, 1)
    tot = cum[:, -1]
    x = (cum <= (st["us"].double() * tot)[:, None]).sum(1)
    lastpos = V - 1 - torch.argmax((res.flip(1) > 0).int(), 1)
    x = torch.minimum(x, lastpos)
    x = torch.where(tot > 0, x, torch.full_like(x, -1))
    col = torch.arange(k + 1, device="cuda")[None]
    pad = torch.cat([draft, draft[:, :1]], 1)
    out = torch.where(col < r[:, None], pad, torch.where(col == r[:, None], x[:, None], torch.full_like(pad, -1)))
    st["tokens"].copy_(out)
    st["count"].copy_(r + 1)


def run(st):
    case = st["case"]
    kind = case["kind"]
    stream = torch.cuda.current_stream()
    if kind == "prompt":
        if own:
            _pkg().attn_prompt(st["q"], st["k"], st["v"], st["out"], st["cu"], stream=stream)
            return st["out"]
        return _plain_prompt(st)
    if kind == "prefix":
        if own:
            st["pages"].attn_prefix(st["layer"], st["q"], st["out"], st["slots"], case["prefix"], st["scratch"],
                                    st["status"], stream=stream)
            return [st["out"], st["status"]]
        return [_plain_prefix(st), st["status"]]
    if kind == "fork":
        _restore(st)
        if own:
            st["pages"].fork(st["src"], st["dst"], st["work"], st["status"][:1], stream=stream)
            st["pages"].reserve(st["slots"], st["new"], st["work"], st["status"][1:], stream=stream)
        else:
            _plain_fork(st)
        return [st["k"], st["v"], st["refs"], st["tables"], st["lens"], st["status"]]
    if kind == "compact":
        _restore(st)
        if own:
            st["pages"].compact(st["work"], st["status"], stream=stream)
        else:
            _plain_compact(st)
        return [st["k"], st["v"], st["refs"], st["tables"], st["lens"], st["status"]]
    if kind == "append":
        if own:
            st["pages"].append(st["layer"], st["slot"], st["pos"], st["qi"], st["ki"], st["vi"], st["cos"], st["sin"],
                               st["qo"], st["ko"], st["vo"], st["status"], stream=stream)
        else:
            _plain_append(st)
        return [st["qo"], st["ko"], st["vo"], st["k"], st["v"], st["status"]]
    if own:
        _pkg().spec_verify(st["p"], st["q"], st["draft"], st["nd"], st["ua"], st["us"], st["tokens"], st["count"],
                           stream=stream)
    else:
        _plain_verify(st)
    return [st["tokens"], st["count"]]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    e = 2 if case.get("f16") else 4
    if kind == "prompt":
        lens = [int(x) for x in case["lens"].split(",")]
        return {"bytes": e * D * sum(lens) * (2 * case["H"] + 2 * case["Hkv"]),
                "flops": 4 * D * case["H"] * sum(x * (x + 1) // 2 for x in lens)}
    if kind == "prefix":
        mean = (min(case["nq"], case["own"]) + case["own"]) / 2
        kv = case["prefix"] + case["n"] * mean
        rows = case["n"] * case["nq"] * case["H"]
        return {"bytes": int(e * D * (2 * case["Hkv"] * kv + 2 * rows)),
                "flops": int(4 * D * rows * (case["prefix"] + mean))}
    if kind == "fork":
        part = case["len"] % case["page"] if case["new"] else 0
        row = e * D * case["layers"] * case["Hkv"] * 2
        used = -(-case["len"] // case["page"])
        return {"bytes": 2 * part * row * case["parents"] * case["children"]
                + 8 * used * case["parents"] * (1 + case["children"]), "flops": 0}
    if kind == "compact":
        live = case["slots"] * (case["len"] / 2 / case["page"] + 0.5) * 0.9
        moved = live * (1 - live / case["pages"])
        row = e * D * case["layers"] * case["Hkv"] * 2 * case["page"]
        return {"bytes": int(2 * moved * row + 4 * case["pages"]), "flops": 0}
    if kind == "append":
        h = case["H"] + 2 * case["Hkv"]
        return {"bytes": case["T"] * D * (4 * h + e * h + e * 2 * case["Hkv"]),
                "flops": case["T"] * D * 3 * (case["H"] + case["Hkv"])}
    rows = 1 if case["point"] else 2
    return {"bytes": 4 * case["n"] * case["V"] * rows, "flops": 2 * case["n"] * case["V"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "prompt":
        H, G = case["H"], case["H"] // case["Hkv"]
        out = torch.zeros((sum(st["lens"]), H, D), dtype=torch.float64, device="cuda")
        at = 0
        for L in st["lens"]:
            for h in range(H):
                q = st["q"][at:at + L, h].double()
                k = st["k"][at:at + L, h // G].double()
                v = st["v"][at:at + L, h // G].double()
                for a in range(0, L, 2048):
                    b = min(L, a + 2048)
                    s = (q[a:b] @ k[:b].T) / math.sqrt(D)
                    seen = torch.ones_like(s).tril(a)
                    w = torch.exp(s - torch.where(seen > 0, s, -math.inf).amax(1, keepdim=True)) * seen
                    out[at + a:at + b, h] = (w @ v[:b]) / w.sum(1, keepdim=True)
            at += L
        return out
    if kind == "prefix":
        n, nq, H, G, page = case["n"], case["nq"], case["H"], case["H"] // case["Hkv"], case["page"]
        out = torch.zeros((n, nq, H, D), dtype=torch.float64, device="cuda")
        tables, lens, slots = st["tables"].tolist(), st["lens"].tolist(), st["slots"].tolist()
        for b, s in enumerate(slots):
            L = lens[s]
            ids = torch.tensor(tables[s][:(L + page - 1) // page], device="cuda")
            k = st["k"][ids, st["layer"]].double().transpose(0, 1).reshape(case["Hkv"], -1, D)[:, :L]
            v = st["v"][ids, st["layer"]].double().transpose(0, 1).reshape(case["Hkv"], -1, D)[:, :L]
            for t in range(nq):
                m = L - nq + 1 + t
                if m <= 0:
                    continue
                q = st["q"][b, t].double().view(case["Hkv"], G, D)
                w = torch.softmax(q @ k[:, :m].transpose(1, 2) / math.sqrt(D), -1)
                out[b, t] = (w @ v[:, :m]).reshape(H, D)
        return [out, None]
    if kind == "append":
        pos = st["pos"].long()
        c, s = st["cos"].double()[pos].unsqueeze(1), st["sin"].double()[pos].unsqueeze(1)
        rot = []
        for x in (st["qi"].double(), st["ki"].double()):
            y = torch.empty_like(x)
            y[..., :64] = x[..., :64] * c - x[..., 64:] * s
            y[..., 64:] = x[..., :64] * s + x[..., 64:] * c
            rot.append(y)
        k, v, page = st["k"].double(), st["v"].double(), case["page"]
        tables = st["tables"].tolist()
        where = [(tables[a][b // page], b % page) for a, b in zip(st["slot"].tolist(), st["pos"].tolist())]
        pg, at = torch.tensor([w[0] for w in where], device="cuda"), torch.tensor([w[1] for w in where], device="cuda")
        k[pg, st["layer"], :, at] = rot[1]
        v[pg, st["layer"], :, at] = st["vi"].double()
        return [rot[0], rot[1], st["vi"].double(), k, v, None]
    if kind == "verify":
        n, k = case["n"], case["k"]
        toks = np.full((n, k + 1), -1, np.int64)
        cnt = np.zeros(n, np.int64)
        draft, nd = st["draft"].tolist(), st["nd"].tolist()
        ua, us = st["ua"].double().tolist(), st["us"].double().tolist()
        for b in range(n):
            r = 0
            while r < nd[b]:
                x = draft[b][r]
                qx = 1.0 if st["q"] is None else float(st["q"][b, r, x])
                if not ua[b][r] * qx < float(st["p"][b, r, x]):
                    break
                toks[b, r] = x
                r += 1
            mass = st["p"][b, r].cpu().numpy().astype(np.float64)
            if r < nd[b]:
                if st["q"] is None:
                    rest = mass.copy()
                    rest[draft[b][r]] = 0.0
                else:
                    rest = np.maximum(mass - st["q"][b, r].cpu().numpy().astype(np.float64), 0.0)
                if rest.sum() > 0:
                    mass = rest
            cum = np.cumsum(mass)
            if cum[-1] > 0:
                x = int(np.searchsorted(cum, us[b] * cum[-1], side="right"))
                toks[b, r] = min(x, int(np.nonzero(mass)[0][-1]))
            cnt[b] = r + 1
        return [torch.tensor(toks, dtype=torch.int32, device="cuda"), torch.tensor(cnt, dtype=torch.int32, device="cuda")]
    return None                          # pages are moved, not computed
