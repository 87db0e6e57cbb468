"""The 8-bit paged cache and the beam search operators: what is measured, and their plain forms.

A case is one pass as a serving loop makes it. `run` computes it with elementary torch operations, or
through the library's own entry points where `own` is true.

kind "store"  RoPE and the store of new tokens in an 8-bit cache, then the blocks that they touched read
              back (sllm_cuda_kv8_append, sllm_cuda_kv8_read)
kind "read"   whole conversations read back from an 8-bit cache (sllm_cuda_kv8_read)
kind "attn8"  decode attention over an 8-bit cache (sllm_cuda_attn_kv8)
kind "beam"   a beam search's selection over beams and vocabulary, and the reordering of the beams'
              tables (sllm_cuda_beam_select, sllm_cuda_kv_fork)

The 8-bit cache: codes -127 .. 127 and one scale for 16 tokens of a head; a value is code * scale.
"""
import importlib
import math

import numpy as np
import torch

own = False

D = 128                       # the head dimension of every model the library runs
BLOCK = 16                    # tokens that share a scale
SCALE = 1.0 / math.sqrt(D)
LEAST = 2.0 ** -100           # the least scale of a block that is not all zeros


def listed():
    return [
        # one decode step's new tokens of a batch of 16: latency
        {"name": "store_step_f16", "kind": "store", "f16": True, "H": 20, "Hkv": 5, "T": 16, "slots": 16,
         "page": 16, "layers": 2},
        # a chunk of a prompt for each of three conversations, f32 outside the cache
        {"name": "store_chunk_f32", "kind": "store", "f16": False, "H": 20, "Hkv": 5, "T": 300, "slots": 3,
         "page": 32, "layers": 2},
        # a prefill's tokens through the 64/8 heads of the 80-layer model
        {"name": "store_prompt_f16", "kind": "store", "f16": True, "H": 64, "Hkv": 8, "T": 4099, "slots": 5,
         "page": 64, "layers": 1},
        # a conversation's earlier turns for the attention of its next prompt, f32
        {"name": "read_turns_f32", "kind": "read", "f16": False, "Hkv": 5, "T": 777, "slots": 2, "page": 16, "layers": 2},
        # a long document's keys and values
        {"name": "read_document_f16", "kind": "read", "f16": True, "Hkv": 8, "T": 32768, "slots": 1, "page": 64,
         "layers": 1},
        # one short conversation, f32 queries: the smallest call
        {"name": "attn8_one_f32", "kind": "attn8", "f16": False, "H": 20, "Hkv": 5, "n": 1, "nq": 1, "len": 320,
         "page": 16, "layers": 2},
        # a decode step of 16 conversations, small pages
        {"name": "attn8_batch_f16", "kind": "attn8", "f16": True, "H": 20, "Hkv": 5, "n": 16, "nq": 1, "len": 4000,
         "page": 16, "layers": 1},
        # 32 conversations with three drafted tokens each to score
        {"name": "attn8_draft_f16", "kind": "attn8", "f16": True, "H": 64, "Hkv": 8, "n": 32, "nq": 4, "len": 4096,
         "page": 64, "layers": 1},
        # one conversation over a long document
        {"name": "attn8_long_f16", "kind": "attn8", "f16": True, "H": 64, "Hkv": 8, "n": 1, "nq": 1, "len": 131072,
         "page": 128, "layers": 1},
        # a full batch of 64 through the 64/8 heads
        {"name": "attn8_full_f16", "kind": "attn8", "f16": True, "H": 64, "Hkv": 8, "n": 64, "nq": 1, "len": 8192,
         "page": 64, "layers": 1},
        # one request with four beams over the 128256-word vocabulary
        {"name": "beam_one", "kind": "beam", "n": 1, "B": 4, "V": 128256, "done": 0.0, "masked": 0.0, "first": False,
         "len": 300, "page": 16},
        # 32 requests of eight beams, some of them finished
        {"name": "beam_batch", "kind": "beam", "n": 32, "B": 8, "V": 128256, "done": 0.1, "masked": 0.0, "first": False,
         "len": 2000, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice([(20, 5), (64, 8), (8, 1), (4, 4), (6, 2), (14, 2)])
    kind = rng.choice(["store", "read", "attn8", "attn8", "beam"])
    f16 = rng.random() < 0.6
    page = rng.choice([16, 32, 64, 128])
    if kind == "store":
        return {"kind": kind, "f16": f16, "H": heads[0], "Hkv": heads[1], "T": _log(rng, 1, 4000),
                "slots": rng.randint(1, 16), "page": page, "layers": rng.randint(1, 3)}
    if kind == "read":
        return {"kind": kind, "f16": f16, "Hkv": heads[1], "T": _log(rng, 1, 32000), "slots": rng.randint(1, 12),
                "page": page, "layers": rng.randint(1, 2)}
    if kind == "attn8":
        n = _log(rng, 1, 64)
        nq = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        most = min(60000, 4000000 // (n * heads[1] * (1 if f16 else 2)) // (1 if nq < 3 else 2))
        return {"kind": kind, "f16": f16, "H": heads[0], "Hkv": heads[1], "n": n, "nq": nq, "len": _log(rng, nq, most),
                "page": page, "layers": rng.randint(1, 2)}
    return {"kind": kind, "n": _log(rng, 1, 32), "B": rng.choice([1, 2, 3, 4, 5, 6, 8]), "V": _log(rng, 2, 128256),
            "done": rng.choice([0.0, 0.0, 0.2, 1.0]), "masked": rng.choice([0.0, 0.0, 0.5, 0.999]),
            "first": rng.random() < 0.2, "len": _log(rng, 1, 2000), "page": page}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dt(case):
    return torch.float16 if case["f16"] else torch.float32


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _pkg():
    return importlib.import_module("saphira-llm_b200")


def _pool(g, shape):
    """Codes and scales of one pool in use: what quantised keys or values look like."""
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    for i in range(0, shape[0], 4096):          # (a large pool's random numbers in f32 would not fit beside it)
        part = torch.randn(codes[i:i + 4096].shape, generator=g, device="cuda")
        codes[i:i + 4096] = part.mul_(42.0).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.randn(shape[:3] + (shape[3] // BLOCK,), generator=g, device="cuda").mul_(0.3).exp_().mul_(1 / 42)
    return codes, scales


def _cache(case, seed, lens, n_pages=None):
    """A cache whose slots hold `lens` tokens, in pages of no order."""
    page, r = case["page"], np.random.default_rng(seed + 7)
    used = [(x + page - 1) // page for x in lens]
    n_pages = n_pages or sum(used) + 5
    ids = r.permutation(n_pages)
    tab = np.full((len(lens), max(used) + 1), -1, np.int64)
    refs = np.zeros(n_pages, np.int64)
    at = 0
    for s, u in enumerate(used):
        tab[s, :u] = ids[at:at + u]
        refs[tab[s, :u]] = 1
        at += u
    shape = (n_pages, case["layers"], case["Hkv"], page, D)
    g = _gen(seed + 3)
    (k, ks), (v, vs) = _pool(g, shape), _pool(g, shape)
    return {"case": case, "layer": case["layers"] - 1, "k": k, "v": v, "ks": ks, "vs": vs, "refs": _i32(refs.tolist()),
          "tables": _i32(tab.tolist()), "lens": _i32(list(lens)), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _handle(st):
    if own:
        st["pages"] = _pkg().KvPages(st["k"], st["v"], st["refs"], st["tables"], st["lens"], st["ks"], st["vs"])
    return st


def _spread(total, parts, r):
    return np.bincount(np.sort(r.integers(0, parts, total)), minlength=parts)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    r = np.random.default_rng(seed)
    if kind == "store":
        H, Hkv, T, S, page = case["H"], case["Hkv"], case["T"], case["slots"], case["page"]
        cnt = _spread(T, S, r)
        past = r.integers(0, 2 * page + 1, S)
        st = _cache(case, seed, [int(x) for x in cnt + past], T // page + 3 * S + 3)
        slot = np.repeat(np.arange(S), cnt)
        pos = np.concatenate([past[s] + np.arange(cnt[s]) for s in range(S)])
        # the blocks that the new tokens touch, from their first tokens on; padded with tokens of no slot
        first = past // BLOCK * BLOCK
        seen = [np.arange(first[s], past[s] + cnt[s]) if cnt[s] else np.arange(0) for s in range(S)]
        n_read = T + S * (BLOCK - 1)
        rslot, rpos = np.full(n_read, -1, np.int64), np.zeros(n_read, np.int64)
        back = np.concatenate(seen)
        rslot[:len(back)] = np.repeat(np.arange(S), [len(x) for x in seen])
        rpos[:len(back)] = back
        n_ctx = int((cnt + past).max())
        ang = np.arange(n_ctx)[:, None] * (500000.0 ** (-2.0 * np.arange(D // 2) / D))[None]
        # the projections' outputs, one array; tokens differ in magnitude
        qkv = torch.randn((T, H + 2 * Hkv, D), generator=g, device="cuda")
        qkv *= torch.randn((T, 1, 1), generator=g, device="cuda").mul_(0.3).exp_()
        dt = _dt(case)
        st.update({"slot": _i32(slot.tolist()), "pos": _i32(pos.tolist()), "rslot": _i32(rslot.tolist()),
                   "rpos": _i32(rpos.tolist()),
                   "cos": torch.tensor(np.cos(ang), dtype=torch.float32, device="cuda"),
                   "sin": torch.tensor(np.sin(ang), dtype=torch.float32, device="cuda"), "qi": qkv[:, :H],
                   "ki": qkv[:, H:H + Hkv], "vi": qkv[:, H + Hkv:], "qo": torch.empty((T, H, D), dtype=dt, device="cuda"),
                   "ko": torch.zeros((n_read, Hkv, D), dtype=dt, device="cuda"),
                   "vo": torch.zeros((n_read, Hkv, D), dtype=dt, device="cuda")})
        return _handle(st)
    if kind == "read":
        S, T = case["slots"], case["T"]
        cnt = _spread(T, S, r)
        st = _cache(case, seed, [int(x) for x in cnt])
        dt = _dt(case)
        st.update({"rslot": _i32(np.repeat(np.arange(S), cnt).tolist()),
                   "rpos": _i32(np.concatenate([np.arange(c) for c in cnt]).tolist()),
                   "ko": torch.empty((T, case["Hkv"], D), dtype=dt, device="cuda"),
                   "vo": torch.empty((T, case["Hkv"], D), dtype=dt, device="cuda")})
        return _handle(st)
    if kind == "attn8":
        n, nq, H, dt = case["n"], case["nq"], case["H"], _dt(case)
        lens = r.integers(nq, case["len"] + 1, n + 2)
        if n == 1:
            lens[:] = nq                                     # (the slots that this call does not name)
        slots = r.permutation(n + 2)[:n]
        if n == 1:
            lens[slots[0]] = case["len"]
        st = _cache(case, seed, [int(x) for x in lens])
        st.update({"seen": int(lens[slots].max()), "slots": _i32(slots.tolist()),
                   "q": (torch.randn((n, nq, H, D), generator=g, device="cuda") * 1.5).to(dt),
                   "out": torch.empty((n, nq, H, D), dtype=dt, device="cuda")})
        _handle(st)
        if own:
            st["work"] = torch.empty(st["pages"].attn8_work_bytes(n, nq, H), dtype=torch.uint8, device="cuda")
        return st
    # a beam search: the beams of a request share its prompt's pages and have one or more of their own
    n, B, V, page = case["n"], case["B"], case["V"], case["page"]
    plen = case["len"]
    full, S = plen // page, n * B
    tail = r.integers(0, page + 1, n)                        # tokens since: the same for a request's beams
    more = ((plen % page + tail) + page - 1) // page
    n_pages = n * full + 2 * S + 5
    ids = r.permutation(n_pages)
    tab = np.full((S, full + 3), -1, np.int64)
    lens = np.zeros(S, np.int64)
    refs = np.zeros(n_pages, np.int64)
    at = 0
    for i in range(n):
        head = ids[at:at + full]
        at += full
        for b in range(B):
            tab[i * B + b, :full] = head
            tab[i * B + b, full:full + more[i]] = ids[at:at + more[i]]
            at += more[i]
            lens[i * B + b] = plen + tail[i]
            np.add.at(refs, tab[i * B + b, :full + more[i]], 1)
    shape = (n_pages, 1, 1, page, D)
    # logits of beams that read nearly the same text; some words forbidden
    base = torch.randn((n, 1, V), generator=g, device="cuda") * 2.5
    logits = base + torch.randn((n, B, V), generator=g, device="cuda") * 1.2
    if case["masked"] > 0:
        logits.masked_fill_(torch.rand((n, 1, V), generator=g, device="cuda") < case["masked"], -math.inf)
    score = torch.randn((n, B), generator=g, device="cuda") * 1.5 - 20.0
    if case["first"]:
        score[:, 0] = 0.0
        score[:, 1:] = -math.inf
    done = (torch.rand((n, B), generator=g, device="cuda") < case["done"]).to(torch.int32)
    st = {"case": case, "logits": logits, "score": score, "done": done, "eos": V // 2,
          "k": torch.zeros(shape, dtype=torch.int8, device="cuda"), "v": torch.zeros(shape, dtype=torch.int8, device="cuda"),
          "ks": torch.zeros(shape[:3] + (page // BLOCK,), device="cuda"),
          "vs": torch.zeros(shape[:3] + (page // BLOCK,), device="cuda"), "refs": _i32(refs.tolist()),
          "tables": _i32(tab.tolist()), "lens": _i32(lens.tolist()), "slots": _i32(r.permutation(S).tolist()),
          "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    order = st["slots"].long()                               # slot slots[i] is beam i
    for name in ("tables", "lens"):
        t = torch.empty_like(st[name])
        t[order] = st[name]
        st[name] = t
    st["saved"] = [st[x].clone() for x in ("refs", "tables", "lens")]
    for name, dt in (("score_out", torch.float32), ("parent", torch.int32), ("token", torch.int32),
                     ("done_out", torch.int32), ("src", torch.int32)):
        st[name] = torch.empty((n, B), dtype=dt, device="cuda")
    _handle(st)
    if own:
        st["work"] = torch.empty(st["pages"].work_bytes(), dtype=torch.uint8, device="cuda")
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_store(st):
    """A block's scale grows where a new token needs it, and its earlier tokens' codes follow."""
    page, layer = st["case"]["page"], st["layer"]
    pos, slot = st["pos"].long(), st["slot"].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def rope(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    st["qo"].copy_(rope(st["qi"]))
    width = st["tables"].shape[1] * page // BLOCK
    blocks, of = torch.unique(slot * width + pos // BLOCK, return_inverse=True)       # [nb], token -> its block
    bslot, bidx = blocks // width, blocks % width
    ids, place = st["tables"][bslot, bidx * BLOCK // page].long(), bidx % (page // BLOCK)
    row = torch.arange(BLOCK, device="cuda")
    first = torch.full_like(blocks, BLOCK).scatter_reduce(0, of, pos % BLOCK, "amin")   # rows before it hold older tokens
    rows = place[:, None] * BLOCK + row[None]                                           # [nb, 16] rows of the page
    for x, codes, scales in ((rope(st["ki"]), st["k"], st["ks"]), (st["vi"], st["v"], st["vs"])):
        most = x.abs().amax(-1)                                                       # [T, Hkv]
        top = torch.zeros((blocks.shape[0], x.shape[1]), device="cuda").scatter_reduce(
            0, of[:, None].expand(-1, x.shape[1]), most, "amax")
        old = torch.where(first[:, None] > 0, scales[ids, layer, :, place], torch.zeros_like(top))
        seven = torch.full_like(top, 127.0)
        grows = top > old * seven
        new = torch.where(grows, torch.clamp(torch.div(top, seven), min=LEAST), old)
        inv = torch.where(new > 0, torch.div(torch.ones_like(new), new), torch.zeros_like(new))
        was = codes[ids[:, None], layer, :, rows]                                     # [nb, 16, Hkv, 128]
        again = torch.round(was.float() * (old * inv)[:, None, :, None]).to(torch.int8)
        keep = (row[None] < first[:, None])[:, :, None, None] & grows[:, None, :, None]
        codes[ids[:, None], layer, :, rows] = torch.where(keep, again, was)
        scales[ids, layer, :, place] = new
        mine = torch.clamp(torch.round(x * inv[of][..., None]), -127, 127).to(torch.int8)
        codes[ids[of], layer, :, pos % page] = mine
    st["status"].zero_()


def _plain_read(st):
    page, layer = st["case"]["page"], st["layer"]
    slot, pos = st["rslot"].long(), st["rpos"].long()
    live = (slot >= 0)[:, None, None]                        # (padding is left as it is)
    ids = torch.where(slot >= 0, st["tables"][slot.clamp(min=0), pos // page].long(), 0)
    for codes, scales, out in ((st["k"], st["ks"], st["ko"]), (st["v"], st["vs"], st["vo"])):
        s = scales[ids, layer, :, pos % page // BLOCK]
        x = codes[ids, layer, :, pos % page].float() * s[..., None]
        out.copy_(torch.where(live, x.to(out.dtype), out))
    st["status"].zero_()


def _plain_attn8(st):
    case, out = st["case"], st["out"]
    H, Hkv, page, n, nq, layer = case["H"], case["Hkv"], case["page"], case["n"], case["nq"], st["layer"]
    G = H // Hkv
    slots = st["slots"].long()
    m = (st["seen"] + page - 1) // page
    ids = st["tables"][slots].long()[:, :m].clamp(min=0)                              # [n, m]
    j = torch.arange(m * page, device="cuda")
    # query t of a sequence sees its first len - nq + 1 + t tokens
    limit = st["lens"][slots].long()[:, None] - nq + 1 + torch.arange(nq, device="cuda")[None]
    dead = (j[None, None] >= limit[:, :, None])[:, :, None]                           # [n, nq, 1, L]

    def values(codes, scales, h):
        x = codes[:, layer, h][ids].float().view(n, m, page // BLOCK, BLOCK, D)
        return (x * scales[:, layer, h][ids][..., None, None]).view(n, m * page, D)

    for h in range(Hkv):
        q = st["q"][:, :, h * G:(h + 1) * G].float().reshape(n, nq * G, D)
        s = torch.matmul(q, values(st["k"], st["ks"], h).transpose(1, 2)).view(n, nq, G, m * page) * SCALE
        s = s.masked_fill(dead, float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        v = values(st["v"], st["vs"], h).masked_fill((j[None] >= limit[:, -1:])[..., None], 0.0)
        o = torch.matmul(e.view(n, nq * G, m * page), v).view(n, nq, G, D) / e.sum(-1, keepdim=True)
        out[:, :, h * G:(h + 1) * G] = o.to(out.dtype)
    st["status"].zero_()


def _restore(st):
    for name, t in zip(("refs", "tables", "lens"), st["saved"]):
        st[name].copy_(t)


def _plain_beam(st):
    case, V, B = st["case"], st["case"]["V"], st["case"]["B"]
    low = -1e300                                             # stands for a candidate of weight 0; -inf for none
    x = torch.where(st["logits"] < math.inf, st["logits"], -math.inf).double()
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    cand = st["score"].double()[..., None] + (x - lse)
    cand = torch.where(cand > low, cand, low)                # (a NaN too)
    word = torch.arange(V, device="cuda")
    done = (st["done"] != 0)[..., None]
    cand = torch.where(done, torch.where(word == st["eos"], st["score"].double()[..., None].clamp(min=low), -math.inf), cand)
    flat = cand.view(case["n"], B * V)
    row = torch.arange(case["n"], device="cuda")
    for i in range(B):
        at = torch.argmax(flat, 1)                           # the first of equals
        got = flat[row, at]
        flat[row, at] = -math.inf
        st["score_out"][:, i] = torch.where(got > low, got, -math.inf).float()
        st["parent"][:, i] = at // V
        st["token"][:, i] = at % V
    pick = st["parent"].long()
    st["done_out"].copy_(torch.gather(st["done"], 1, pick) | (st["token"] == st["eos"]).int())
    st["src"].copy_(torch.gather(st["slots"].view(case["n"], B), 1, pick))
    # every beam's slot takes its parent's pages, all at once
    page, refs, tab, lens = case["page"], st["refs"], st["tables"], st["lens"]
    src, dst = st["src"].view(-1).long(), st["slots"].long()
    col = torch.arange(tab.shape[1], device="cuda")[None]
    rows, old = tab[src], tab[dst]
    used = col < ((lens[src] + page - 1) // page)[:, None]
    was = col < ((lens[dst] + page - 1) // page)[:, None]
    refs.index_add_(0, torch.where(used, rows, 0).reshape(-1).long(), used.reshape(-1).int())
    refs.index_add_(0, torch.where(was, old, 0).reshape(-1).long(), -was.reshape(-1).int())
    tab[dst] = torch.where(used, rows, old)
    lens[dst] = lens[src]
    st["status"].zero_()


def run(st):
    case = st["case"]
    kind = case["kind"]
    stream = torch.cuda.current_stream()
    if kind == "store":
        if own:
            st["pages"].append8(st["layer"], st["slot"], st["pos"], st["qi"], st["ki"], st["vi"], st["cos"], st["sin"],
                                st["qo"], status=st["status"], stream=stream)
            st["pages"].read8(st["layer"], st["rslot"], st["rpos"], st["ko"], st["vo"], st["status"], stream=stream)
        else:
            _plain_store(st)
            _plain_read(st)
        return [st["qo"], st["ko"], st["vo"], st["ks"], st["vs"], st["status"]]
    if kind == "read":
        if own:
            st["pages"].read8(st["layer"], st["rslot"], st["rpos"], st["ko"], st["vo"], st["status"], stream=stream)
        else:
            _plain_read(st)
        return [st["ko"], st["vo"], st["status"]]
    if kind == "attn8":
        if own:
            st["pages"].attn8(st["layer"], st["q"], st["out"], st["slots"], st["work"], st["status"], stream=stream)
        else:
            _plain_attn8(st)
        return [st["out"], st["status"]]
    _restore(st)
    if own:
        _pkg().beam_select(st["logits"], st["score"], st["score_out"], st["parent"], st["token"], done=st["done"],
                           eos=st["eos"], done_out=st["done_out"], slots=st["slots"], src=st["src"], status=st["status"],
                           stream=stream)
        st["pages"].fork(st["src"].view(-1), st["slots"], st["work"], st["status"], stream=stream)
    else:
        _plain_beam(st)
    return [st["parent"], st["token"], st["score_out"], st["done_out"], st["src"], st["refs"], st["tables"], st["lens"],
            st["status"]]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    e = 2 if case.get("f16") else 4
    if kind == "store":
        rows = case["T"] + min(case["slots"], case["T"]) * 7.5     # read back: with the older tokens of the first blocks
        h = case["H"] + 2 * case["Hkv"]
        return {"bytes": int(D * (case["T"] * (4 * h + e * case["H"] + 2 * case["Hkv"]) + rows * 2 * case["Hkv"] * (1 + e))),
                "flops": int(case["T"] * D * (3 * (case["H"] + case["Hkv"]) + 3 * 2 * case["Hkv"]))}
    if kind == "read":
        return {"bytes": int(case["T"] * 2 * case["Hkv"] * (D * (1 + e) + 4 / BLOCK)), "flops": case["T"] * 2 * case["Hkv"] * D}
    if kind == "attn8":
        mean = case["len"] if case["n"] == 1 else (case["nq"] + case["len"]) / 2
        rows = case["n"] * case["nq"] * case["H"]
        return {"bytes": int(case["n"] * mean * case["Hkv"] * 2 * (D + 4 / BLOCK) + 2 * e * D * rows),
                "flops": int(4 * D * rows * mean)}
    live = 1.0 - case["done"]
    if case["first"]:
        live /= case["B"]
    table = 4 * case["n"] * case["B"] * (case["len"] // case["page"] + 1)
    return {"bytes": int(4 * case["n"] * case["B"] * case["V"] * live) + 3 * table,
            "flops": int(3 * case["n"] * case["B"] * case["V"] * live)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "store":
        pos = st["pos"].long()
        c, s = st["cos"].double()[pos].unsqueeze(1), st["sin"].double()[pos].unsqueeze(1)
        q = st["qi"].double()
        rot = torch.cat([q[..., :64] * c - q[..., 64:] * s, q[..., :64] * s + q[..., 64:] * c], -1)
        return [rot, None, None, None, None, None]           # codes: a rounding step either way is no error
    if kind == "read":
        ids = st["tables"][st["rslot"].long(), st["rpos"].long() // case["page"]].long()
        at = st["rpos"].long() % case["page"]
        return [codes[ids, st["layer"], :, at].double() * sc[ids, st["layer"], :, at // 16].double()[..., None]
                for codes, sc in ((st["k"], st["ks"]), (st["v"], st["vs"]))] + [None]
    if kind == "attn8":
        n, nq, H, Hkv, page = case["n"], case["nq"], case["H"], case["Hkv"], case["page"]
        out = torch.zeros((n, nq, H, D), dtype=torch.float64, device="cuda")
        tables, lens, slots = st["tables"].tolist(), st["lens"].tolist(), st["slots"].tolist()
        for b, s in enumerate(slots):
            L = lens[s]
            ids = torch.tensor(tables[s][:(L + page - 1) // page], device="cuda")
            kv = []
            for codes, sc in ((st["k"], st["ks"]), (st["v"], st["vs"])):
                x = codes[ids, st["layer"]].double() * sc[ids, st["layer"]].double().repeat_interleave(16, -1)[..., None]
                kv.append(x.transpose(0, 1).reshape(Hkv, -1, D)[:, :L])
            for t in range(nq):
                m = L - nq + 1 + t
                q = st["q"][b, t].double().view(Hkv, H // Hkv, D)
                w = torch.softmax(q @ kv[0][:, :m].transpose(1, 2) / math.sqrt(D), -1)
                out[b, t] = (w @ kv[1][:, :m]).reshape(H, D)
        return [out, None]
    n, B, V = case["n"], case["B"], case["V"]
    found = torch.empty((n, B), dtype=torch.float64, device="cuda")
    done, score = st["done"].tolist(), st["score"].double().tolist()
    for i in range(n):
        lists = []
        for b in range(B):
            if done[i][b]:
                lists.append(torch.tensor([score[i][b]], dtype=torch.float64, device="cuda"))
            else:
                lp = score[i][b] + torch.log_softmax(st["logits"][i, b].double(), -1)
                lists.append(torch.where(torch.isnan(lp), -math.inf, lp))
        found[i] = torch.sort(torch.cat(lists), descending=True).values[:B]
    return [None, None, found, None, None, None, None, None, None]
