"""The operators around attention that serving calls step by step, as sizes to time and to check.

rotary       rotary positions on q and k, with their table for long contexts and their gradient
append       new K and V rows quantised to 4 bits into the pages of a cache
attend       attention of a few new tokens over such a cache, with or without each token's accumulated weight
evict        the cache cut back to a budget by that weight, after a step or a prompt has been appended

With `own` false every pass is computed in plain torch operations in 32 bits; with `own` true it is the calls a
program makes of this library.  A record of one token and head is, in bytes: D / 2 of K codes, D / 2 of V codes,
then for K and for V a (scale, minimum) pair of 16-bit numbers per group of 32 dims.  The sizes are this
repository's head dimensions, heads and lengths, or generic ones.
"""
import math
import os
import sys

import torch

own = False
_mods = None
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_HEADS = 8   # K/V heads where a case does not say


def _library():
    global _mods
    if _mods is None:
        pkg = os.path.join(os.getcwd(), "ascend-rsfa_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from ascend_rsfa import kv_cache, rotary
        _mods = (rotary, kv_cache)
    return _mods


# ------------------------------------------------------------------ cases

def _rotary(name, B, Hq, Hk, S, D, R, dtype, interleaved=False, layout="bhsd", scaling="none", factor=1.0,
            first=0, train=False, table=False):
    c = {"op": "rotary", "B": B, "Hq": Hq, "Hk": Hk, "S": S, "D": D, "R": R, "dtype": dtype, "interleaved": interleaved,
         "layout": layout, "scaling": scaling, "factor": factor, "first": first, "train": train, "table": table}
    return dict(c, name=name) if name else c


def _append(name, B, Hk, S, D, page, dtype, held, ragged=False):
    c = {"op": "append", "B": B, "Hk": Hk, "S": S, "D": D, "page": page, "dtype": dtype, "held": held, "ragged": ragged}
    return dict(c, name=name) if name else c


def _attend(name, B, Hq, Hk, S, D, page, dtype, longest, ragged=False, weights=False):
    c = {"op": "attend", "B": B, "Hq": Hq, "Hk": Hk, "S": S, "D": D, "page": page, "dtype": dtype, "longest": longest,
         "ragged": ragged, "weights": weights}
    return dict(c, name=name) if name else c


def _evict(name, B, Hk, D, page, dtype, budget, fresh, recent):
    c = {"op": "evict", "B": B, "Hk": Hk, "D": D, "page": page, "dtype": dtype, "budget": budget, "fresh": fresh,
         "recent": recent}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One new token of one sequence: latency is all there is.
        _rotary("rotary_token", 1, 32, 8, 1, 128, 128, "bf16", first=700),
        # Q and K of the repository's 4096-token configuration, whole heads, half layout.
        _rotary("rotary_prompt", 16, 16, 16, 4096, 128, 128, "bf16"),
        # A training step on a ragged length straight from a [B, S, H, D] projection: part of the head, interleaved
        # pairs, shared K heads, both directions.
        _rotary("rotary_train", 8, 32, 8, 1000, 128, 64, "fp16", interleaved=True, layout="bshd", train=True),
        # A context that has just grown past its table: the scaled table is made anew and used at its far end.
        _rotary("rotary_far", 1, 32, 8, 4096, 128, 128, "fp16", scaling="yarn", factor=32.0, first=131072 - 4096,
                table=True),
        # One new token for each of 64 sequences in use.
        _append("append_step", 64, 8, 1, 128, 64, "fp16", 1000),
        # Prompts of different lengths as one padded batch.
        _append("append_prompts", 8, 8, 4096, 128, 64, "bf16", 0, ragged=True),
        # The next token of a single short sequence.
        _attend("attend_token", 1, 32, 8, 1, 128, 64, "fp16", 500),
        # A serving batch of ragged lengths, four query heads to a K/V head.
        _attend("attend_batch", 64, 32, 8, 1, 128, 64, "fp16", 8192, ragged=True),
        # One long document, eight query heads to a K/V head, the weights accumulated for a later eviction.
        _attend("attend_long", 2, 64, 8, 1, 128, 128, "bf16", 131072, weights=True),
        # Four tokens to verify per sequence, small heads that share nothing, small pages, weights accumulated.
        _attend("attend_verify_d64", 16, 16, 16, 4, 64, 16, "bf16", 2048, ragged=True, weights=True),
        # A step of a bounded cache: one token in, the lightest one out.
        _evict("evict_step", 32, 8, 128, 64, "fp16", 2048, 1, 256),
        # A prompt cut to a quarter right after it was read.
        _evict("evict_prompt", 4, 8, 128, 64, "bf16", 4096, 12288, 512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "rotary", "append", "attend", "attend", "attend", "evict"))
    dtype = rng.choice(("fp16", "bf16"))
    D = rng.choice((64, 128, 128, 256))
    Hk = rng.choice((1, 2, 4, 8, 16))
    page = rng.choice((16, 32, 64, 128))
    if op == "rotary":
        D = rng.choice((16, 32, 64, 128, 128, 256))
        R = rng.choice((D, D, D // 2, max(2, D // 4 - 2)))
        S = _log(rng, 1, 8192)
        Hq = Hk * rng.choice((1, 2, 4))
        train = rng.random() < 0.3
        cap = max(1, int(1.0e9 / (4 * S * (Hq + Hk) * D * (2 if train else 1))))
        scaling = rng.choice(("none", "linear", "ntk", "yarn", "bands"))
        return _rotary(None, max(1, min(_log(rng, 1, 256), cap)), Hq, Hk, S, D, R, dtype, interleaved=rng.random() < 0.5,
                       layout=rng.choice(("bhsd", "bshd")), scaling=scaling,
                       factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)), first=_log(rng, 1, 30000) - 1,
                       train=train, table=rng.random() < 0.2)
    if op == "append":
        S = _log(rng, 1, 4096)
        B = max(1, min(_log(rng, 1, 256), int(1.3e8 / (S * Hk * D * 4))))
        return _append(None, B, Hk, S, D, page, dtype, _log(rng, 1, 2000) - 1, ragged=S > 1 and rng.random() < 0.5)
    if op == "attend":
        longest = _log(rng, 1, 131072)
        B = max(1, min(_log(rng, 1, 128), int(1.5e8 / (longest * Hk * D))))
        S = rng.choice((1, 1, 1, 2, 5))
        Hq = Hk * rng.choice((1, 2, 3, 4, 8) if S == 1 else (1, 2))
        return _attend(None, B, Hq, Hk, S, D, page, dtype, longest, ragged=rng.random() < 0.6, weights=rng.random() < 0.4)
    budget = _log(rng, 64, 8192)
    fresh = _log(rng, 1, 2 * budget)
    B = max(1, min(_log(rng, 1, 64), int(1.2e8 / ((budget + fresh) * Hk * D))))
    return _evict(None, B, Hk, D, page, dtype, budget, fresh, rng.randint(0, budget))


# ------------------------------------------------------------------ the record's layout

def _k_order(D):
    """Dim held by each nibble of a record's K codes, low nibble of a byte first."""
    G = D // 32
    order = [0] * D
    for w in range(G):
        for c in range(4):
            for j in range(4):
                byte = (w // 4) * 64 + c * 4 * min(G, 4) + 4 * (w % 4) + j
                order[2 * byte] = 32 * w + 8 * c + 2 * j
                order[2 * byte + 1] = 32 * w + 8 * c + 2 * j + 1
    return order


def _v_order(D):
    order = [0] * D
    for g in range(8):
        for w in range(D // 32):
            for j in range(2):
                byte = g * (D // 16) + 2 * w + j
                order[2 * byte] = 32 * w + 4 * g + 2 * j
                order[2 * byte + 1] = 32 * w + 4 * g + 2 * j + 1
    return order


_perm = {}


def _perms(D, device):
    if (D, device) not in _perm:
        k, v = (torch.tensor(o, device=device) for o in (_k_order(D), _v_order(D)))
        _perm[D, device] = (k, v, torch.argsort(k), torch.argsort(v))
    return _perm[D, device]


def _quantise(x, order):
    """[..., D] 16-bit rows to (codes as bytes [..., D / 2], (scale, minimum) pairs as bytes)."""
    D = x.shape[-1]
    f = x.float().unflatten(-1, (D // 32, 32))
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    s = ((hi - lo) * (1.0 / 15.0)).to(x.dtype).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    u = ((f - lo) * inv).round().clamp(0, 15)
    u = u.flatten(-2).to(torch.uint8).index_select(-1, order)
    codes = u[..., 0::2] | (u[..., 1::2] << 4)
    pairs = torch.cat((s, lo), -1).to(x.dtype).flatten(-2).contiguous().view(torch.uint8)
    return codes, pairs


def _records(k, v):
    D = k.shape[-1]
    ko, vo, _, _ = _perms(D, k.device)
    kc, kp = _quantise(k, ko)
    vc, vp = _quantise(v, vo)
    return torch.cat((kc, vc, kp, vp), -1)


def _values(rec, D, dtype):
    """Records [..., 1.25 D] to the K and V values they stand for, in 32 bits."""
    _, _, ki, vi = _perms(D, rec.device)
    G = D // 32
    out = []
    for codes, pairs, inv in ((rec[..., :D // 2], rec[..., D:D + 4 * G], ki), (rec[..., D // 2:D], rec[..., D + 4 * G:], vi)):
        u = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).index_select(-1, inv)
        sm = pairs.contiguous().view(dtype).float().unflatten(-1, (G, 2))
        out.append((u.float().unflatten(-1, (G, 32)) * sm[..., :1] + sm[..., 1:]).flatten(-2))
    return out


def _spread(case, longest):
    """Lengths of the batch: the first as long as can be, the others spread below it."""
    B = case["B"]
    if not case.get("ragged"):
        return [longest] * B
    return [longest] + [1 + int((longest - 1) * ((b * 0.6180339887) % 1.0)) for b in range(1, B)]


# ------------------------------------------------------------------ inputs

def _inverse_frequencies(case):
    """Angles per position of the scaled rotation and what its cosines and sines are multiplied with, in 64 bits."""
    R, base, F, L0 = case["R"], 10000.0, case["factor"], 4096.0
    i = torch.arange(R // 2, dtype=torch.float64)
    if case["scaling"] == "ntk" and R > 2:
        base *= F ** (R / (R - 2.0))
    f = base ** (-2.0 * i / R)
    if case["scaling"] == "linear" or (case["scaling"] == "ntk" and R == 2):
        f = f / F
    mul = 1.0
    if case["scaling"] == "yarn":
        at = [R * math.log(L0 / (2 * math.pi * beta)) / (2 * math.log(base)) for beta in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / F * ramp
        mul = 0.1 * math.log(F) + 1.0 if F > 1 else 1.0
    if case["scaling"] == "bands":
        turns = L0 * f / (2 * math.pi)
        share = ((turns - 1.0) / 3.0).clamp(0, 1)
        f = f * share + f / F * (1 - share)
    return f, mul


def _plain_table(case, length, device):
    f, mul = _inverse_frequencies(case)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * f.to(device)
    return torch.stack((angle.cos() * mul, angle.sin() * mul), -1).float()


def _rand(g, shape, dtype, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype) * std


def _prepare_rotary(case, g):
    B, S, D, dtype = case["B"], case["S"], case["D"], _DTYPES[case["dtype"]]
    x = []
    for H in (case["Hq"], case["Hk"], case["Hq"], case["Hk"]):
        t = _rand(g, (B, H, S, D) if case["layout"] == "bhsd" else (B, S, H, D), dtype)
        x.append(t if case["layout"] == "bhsd" else t.transpose(1, 2))
        if len(x) == 2 and not case["train"]:
            break
    start = case["first"] + torch.randint(0, 16, (B, 1), generator=g, device="cuda")
    start[0] = case["first"]
    pos = (start + torch.arange(S, device="cuda")).to(torch.int32)
    length = case["first"] + S + 16
    st = {"q": x[0], "k": x[1], "pos": pos, "length": length}
    if not case["table"]:
        st["table"] = _plain_table(case, length, "cuda")
    if case["train"]:
        st["q"].requires_grad_(), st["k"].requires_grad_()
        st["dq"], st["dk"] = x[2], x[3]
    return st


def _cache(case, g, lengths, room):
    """Pages in random order for `room` tokens of each sequence, the first lengths[b] of them filled."""
    B, Hk, D, P, dtype = case["B"], case["Hk"], case["D"], case["page"], _DTYPES[case["dtype"]]
    n = -(-room // P)
    order = torch.randperm(B * n, generator=g, device="cuda").to(torch.int32)
    kv = torch.zeros((B * n + 1, Hk, P, D * 5 // 4), dtype=torch.uint8, device="cuda")   # the last page is a spare
    flat = kv[:-1].view(B * n, -1)
    per = max(1, int(3.0e7 / (Hk * P * D)))
    for i in range(0, B * n, per):
        m = min(per, B * n - i)
        k, v = (_rand(g, (m, Hk, P, D), dtype) for _ in range(2))
        flat[i:i + m] = _records(k, v).reshape(m, -1)
    return {"kv": kv, "pages": order.view(B, n).contiguous(), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    if op == "rotary":
        return dict(_prepare_rotary(case, g), case=case)
    B, Hk, D, P = case["B"], case["Hk"], case["D"], case["page"]
    if op == "append":
        S = case["S"]
        counts = _spread(case, S)
        st = _cache(case, g, [case["held"] + c for c in counts], case["held"] + S)
        st["k"], st["v"] = (_rand(g, (B, S, Hk, D), dtype).transpose(1, 2) for _ in range(2))
        st["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None
        st["starts"] = torch.full((B,), case["held"], dtype=torch.int32, device="cuda")
    elif op == "attend":
        lengths = [max(n, case["S"]) for n in _spread(case, case["longest"])]
        st = _cache(case, g, lengths, max(lengths))
        st["q"] = _rand(g, (B, case["S"], case["Hq"], D), dtype, 1.5).transpose(1, 2)
        st["longest"] = max(lengths)
        st["weight"] = torch.rand(st["kv"].shape[:3], generator=g, device="cuda") if case["weights"] else None
    else:
        budget, fresh = case["budget"], case["fresh"]
        st = _cache(case, g, [budget + fresh] * B, budget + fresh)
        shape = st["kv"].shape[:3]
        st["k"], st["v"] = (_rand(g, (B, fresh, Hk, D), dtype).transpose(1, 2) for _ in range(2))
        # what a step's attention adds to every token, and what has been added before
        st["gain"] = torch.rand(shape, generator=g, device="cuda").square()
        st["weight"] = torch.rand(shape, generator=g, device="cuda") * 4
        st["position"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
        slot = torch.arange(budget, device="cuda")
        st["position"][st["pages"][:, slot // P].long(), :, (slot % P).expand(B, -1)] = (2 * slot).to(torch.int32)[None, :, None]
        st["positions"] = (2 * budget + torch.arange(fresh, device="cuda", dtype=torch.int32)).expand(B, -1).contiguous()
    return dict(st, case=case)


# ------------------------------------------------------------------ one pass

def _turn(x, cs, R, interleaved):
    f = x.float()
    c, s = cs[..., 0][:, None], cs[..., 1][:, None]
    if interleaved:
        a, b = f[..., 0:R:2], f[..., 1:R:2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = f[..., :R // 2], f[..., R // 2:R]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, f[..., R:]), -1).to(x.dtype)


def _run_rotary(st, case):
    if own:
        rotary, _ = _library()
        table = st["table"] if "table" in st else rotary.rotary_table(
            st["length"], case["R"], scaling=case["scaling"], factor=case["factor"], original_length=4096, device="cuda")
        q, k = rotary.rotary(st["q"], st["k"], table, st["pos"], case["interleaved"])
    else:
        table = st["table"] if "table" in st else _plain_table(case, st["length"], "cuda")
        cs = table[st["pos"]]
        q, k = (_turn(st[n], cs, case["R"], case["interleaved"]) for n in ("q", "k"))
    if not case["train"]:
        return q, k
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
    return q.detach(), k.detach(), dq, dk


def _plain_append(st, case, counts, lengths):
    P, S = case["page"], case["S"] if "S" in case else case["fresh"]
    j = torch.arange(S, device="cuda")
    slot = (lengths - counts)[:, None] + j if counts is not None else lengths[:, None] - S + j
    page = st["pages"].gather(1, (slot // P).clamp(0, st["pages"].shape[1] - 1).long())
    if counts is not None:   # rows of padding go to the spare page
        page = torch.where(j < counts[:, None], page, st["kv"].shape[0] - 1)
    at = (page.long(), slice(None), (slot % P).long())
    st["kv"][at] = _records(st["k"], st["v"]).transpose(1, 2)
    return at


def _plain_read(st, case, n, starts=None):
    P, dtype = case["page"], _DTYPES[case["dtype"]]
    slot = torch.arange(n, device="cuda").expand(case["B"], n)
    if starts is not None:
        slot = slot + starts[:, None]
    seen = (slot < st["lengths"][:, None])[:, :, None, None]
    page = st["pages"].gather(1, (slot // P).clamp(0, st["pages"].shape[1] - 1).long())
    rec = st["kv"][page.long(), :, (slot % P).long()]
    return [torch.where(seen, x, torch.zeros_like(x)).to(dtype).transpose(1, 2).contiguous() for x in _values(rec, case["D"], dtype)]


def _run_append(st, case):
    n = case["S"]
    if own:
        _, cache = _library()
        cache.cache4_append(st["k"], st["v"], st["kv"], st["pages"], st["lengths"], counts=st["counts"])
        return cache.cache4_read(st["kv"], st["pages"], st["lengths"], n, _DTYPES[case["dtype"]], starts=st["starts"])
    _plain_append(st, case, st["counts"], st["lengths"])
    return _plain_read(st, case, n, st["starts"])


def _run_attend(st, case):
    D, S, scale = case["D"], case["S"], 1.0 / math.sqrt(case["D"])
    if own:
        _, cache = _library()
        o = cache.cache4_attention(st["q"], st["kv"], st["pages"], st["lengths"], scale, weight=st["weight"])
        return o if st["weight"] is None else (o, st["weight"])
    B, Hk, P, N = case["B"], case["Hk"], case["page"], st["longest"]
    slot = torch.arange(N, device="cuda")
    page, off = st["pages"][:, slot // P].long(), (slot % P).expand(B, N)
    k, v = _values(st["kv"][page, :, off], D, _DTYPES[case["dtype"]])          # [B, N, Hk, D]
    q = st["q"].float().unflatten(1, (Hk, case["Hq"] // Hk))                   # [B, Hk, group, S, D]
    s = torch.matmul(q.flatten(2, 3), k.permute(0, 2, 3, 1)).unflatten(2, (-1, S)) * scale
    last = st["lengths"][:, None] - S + torch.arange(S, device="cuda")
    hidden = slot > last[..., None]                                            # [B, S, N]
    s = s.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = v.permute(0, 2, 1, 3)
    v = torch.where((slot < st["lengths"][:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, S)).flatten(1, 2).to(st["q"].dtype)
    if st["weight"] is None:
        return o
    seen = (slot < st["lengths"][:, None])[..., None]
    add = torch.where(seen, p.sum((2, 3)).transpose(1, 2), 0.0)
    at = (torch.where(seen[..., 0], page, st["kv"].shape[0] - 1), slice(None), off)
    st["weight"].index_put_((at[0][:, :, None], torch.arange(Hk, device="cuda"), off[:, :, None]), add, accumulate=True)
    return o, st["weight"]


def _plain_evict(st, case):
    B, Hk, P, budget, recent = case["B"], case["Hk"], case["page"], case["budget"], case["recent"]
    N = budget + case["fresh"]
    slot = torch.arange(N, device="cuda")
    page, off = st["pages"][:, slot // P].long(), (slot % P).expand(B, N)
    w, pos = (st[n][page, :, off].transpose(1, 2) for n in ("weight", "position"))    # [B, Hk, N]
    valid = (slot < st["lengths"][:, None])[:, None].expand(B, Hk, N)
    newest = torch.where(valid, pos, -1).amax(-1, keepdim=True)
    key = torch.where(pos > newest - recent, math.inf, w.clamp(min=0))
    key = torch.where(valid, key, -1.0)
    rank = torch.sort(key, dim=-1, descending=True, stable=True).indices.argsort(-1)
    kept = valid & (rank < budget)
    hole, mover = ~kept[..., :budget], kept & (slot >= budget)
    by_rank = torch.zeros((B, Hk, N + 1), dtype=torch.long, device="cuda")
    by_rank.scatter_(2, torch.where(mover, mover.cumsum(-1) - 1, N), slot.expand(B, Hk, N))
    src = torch.where(hole, by_rank.gather(2, (hole.cumsum(-1) - 1).clamp(min=0)), slot[:budget])
    head = torch.arange(Hk, device="cuda")[None, :, None]
    row = torch.arange(B, device="cuda")[:, None, None]
    frm = (page[row, src], head, src % P)
    to = (page[row, slot[:budget]], head, (slot[:budget] % P).expand(B, Hk, budget))
    for n in ("kv", "weight", "position"):
        st[n][to] = st[n][frm]
    return st["lengths"].clamp(max=budget)


def _run_evict(st, case):
    dtype, budget = _DTYPES[case["dtype"]], case["budget"]
    if own:
        _, cache = _library()
        cache.cache4_append(st["k"], st["v"], st["kv"], st["pages"], st["lengths"], weight=st["weight"],
                            position=st["position"], positions=st["positions"])
        st["weight"] += st["gain"]
        lengths = cache.cache4_evict(st["kv"], st["weight"], st["position"], st["pages"], st["lengths"], budget, case["recent"])
        k, v = cache.cache4_read(st["kv"], st["pages"], lengths, budget, dtype)
    else:
        at = _plain_append(st, case, None, st["lengths"])
        st["weight"][at] = 0.0
        st["position"][at] = st["positions"][..., None]
        st["weight"] += st["gain"]
        lengths = _plain_evict(st, case)
        k, v = _plain_read(dict(st, lengths=lengths), case, budget)
    st["positions"] += case["fresh"]
    return k, v, st["weight"], st["position"], lengths


def run(state):
    case = state["case"]
    return {"rotary": _run_rotary, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[case["op"]](state, case)


# ------------------------------------------------------------------ floors

def work(case):
    B, S, D = case["B"], case.get("S", 0), case["D"]
    if case["op"] == "rotary":
        moved = 2 * 2 * B * (case["Hq"] + case["Hk"]) * S * D
        rows = case["first"] + S + 16 if case["table"] else S
        nbytes = (2 if case["train"] else 1) * (moved + 4 * B * S) + 4 * case["R"] * rows
        return {"bytes": nbytes, "flops": (2 if case["train"] else 1) * 3 * B * (case["Hq"] + case["Hk"]) * S * case["R"]}
    Hk, rec = case["Hk"], D * 5 // 4
    if case["op"] == "append":
        rows = sum(_spread(case, S)) * Hk
        return {"bytes": rows * (4 * D + rec) + rows * rec + B * Hk * S * 4 * D, "flops": 12 * rows * D}
    if case["op"] == "attend":
        lengths = [max(n, S) for n in _spread(case, case["longest"])]
        tokens = sum(lengths) * Hk
        pairs = sum(n * S - S * (S - 1) // 2 for n in lengths) * case["Hq"]
        return {"bytes": tokens * (rec + (8 if case["weights"] else 0)) + 4 * B * case["Hq"] * S * D, "flops": 4 * pairs * D}
    budget, fresh = case["budget"], case["fresh"]
    rows = B * Hk
    moved = min(fresh, budget) * max(1, budget) // (budget + fresh)   # about as many kept rows lie beyond the budget
    nbytes = rows * (fresh * (4 * D + rec + 8) + (budget + fresh) * (8 + 12) + 2 * moved * (rec + 8) + budget * (rec + 4 * D))
    return {"bytes": nbytes, "flops": 12 * rows * (fresh + budget) * D}


# ------------------------------------------------------------------ the definition in 64 bits

def _wide(pairs, dtype):
    return pairs.contiguous().view(dtype).double()


def _exact_rows(rec, D, dtype):
    """Records [n, 1.25 D] to K and V in 64 bits, dim by dim from the layout's formulas."""
    G, half = D // 32, D // 2
    k = torch.empty((rec.shape[0], D), dtype=torch.float64, device=rec.device)
    v = torch.empty_like(k)
    kp, vp = _wide(rec[:, D:D + 4 * G], dtype), _wide(rec[:, D + 4 * G:], dtype)
    for d in range(D):
        w, r = divmod(d, 32)
        kb = (w // 4) * 64 + (r // 8) * 4 * min(G, 4) + (w % 4) * 4 + (r % 8) // 2
        vb = half + (r // 4) * (D // 16) + 2 * w + (r % 4) // 2
        shift = 4 * (d & 1)
        k[:, d] = ((rec[:, kb] >> shift) & 15).double() * kp[:, 2 * w] + kp[:, 2 * w + 1]
        v[:, d] = ((rec[:, vb] >> shift) & 15).double() * vp[:, 2 * w] + vp[:, 2 * w + 1]
    return k, v


def _exact_coded(x):
    """What 16-bit rows read back as, in 64 bits: the scale rounded to the rows' type, the code to the nearest."""
    f = x.double().reshape(*x.shape[:-1], -1, 32)
    lo = f.min(-1, keepdim=True).values
    s = ((f.max(-1, keepdim=True).values - lo) / 15).to(x.dtype).double()
    u = torch.where(s > 0, ((f - lo) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    return (u * s + lo).reshape(x.shape)


def _exact_evict(st, case, D, dtype):
    B, Hk, P, budget, fresh = case["B"], case["Hk"], case["page"], case["budget"], case["fresh"]
    n = budget + fresh
    slot = torch.arange(n, device="cuda")
    weight, position = st["weight"].double(), st["position"].clone()
    new_k, new_v = _exact_coded(st["k"]), _exact_coded(st["v"])
    out = torch.empty((2, B, Hk, budget, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        pages = st["pages"][b].long()[slot // P]
        weight[pages[budget:], :, slot[budget:] % P] = 0
        position[pages[budget:], :, slot[budget:] % P] = st["positions"][b, :, None]
    weight += st["gain"].double()
    for b in range(B):
        pages, off = st["pages"][b].long()[slot // P], slot % P
        for h in range(Hk):
            w, at = weight[pages, h, off], position[pages, h, off]
            # newest positions first, then the heaviest, then the lowest slot
            class_ = torch.where(at > at.max() - case["recent"], math.inf, w)
            chosen = torch.argsort(-class_, stable=True)[:budget]
            chosen = chosen.sort().values
            stay, move = chosen[chosen < budget], chosen[chosen >= budget]
            free = torch.ones(budget, dtype=torch.bool, device="cuda")
            free[stay] = False
            src = slot[:budget].clone()
            src[free] = move
            k, v = _exact_rows(st["kv"][pages, h, off], D, dtype)
            k[budget:], v[budget:] = new_k[b, h], new_v[b, h]
            out[0, b, h], out[1, b, h] = k[src], v[src]
            weight[pages[:budget], h, off[:budget]] = w[src]
            position[pages[:budget], h, off[:budget]] = at[src]
    lengths = st["lengths"].clone()
    lengths[lengths > budget] = budget
    return out[0], out[1], weight, position, lengths


def exact(case, seed):
    st = prepare(case, seed)
    op, D, dtype = case["op"], case["D"], _DTYPES[case["dtype"]]
    if op == "rotary":
        R = case["R"]
        f, mul = _inverse_frequencies(case)
        angle = st["pos"].double()[:, None, :, None] * f.cuda()
        spin = torch.polar(torch.full_like(angle, mul), angle)

        def turn(x, z):
            y = x.detach().double().clone()
            if case["interleaved"]:
                t = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) * z
                y[..., 0:R:2], y[..., 1:R:2] = t.real, t.imag
            else:
                t = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * z
                y[..., :R // 2], y[..., R // 2:R] = t.real, t.imag
            return y

        outs = [turn(st["q"], spin), turn(st["k"], spin)]
        return tuple(outs + [turn(st["dq"], spin.conj()), turn(st["dk"], spin.conj())] if case["train"] else outs)
    if op == "append":
        out = []
        for x in (st["k"], st["v"]):
            y = _exact_coded(x)
            if case["ragged"]:
                y = y * (torch.arange(case["S"], device="cuda") < st["counts"][:, None])[:, None, :, None]
            out.append(y)
        return out
    if op == "evict":
        return _exact_evict(st, case, D, dtype)
    B, Hk, S, P = case["B"], case["Hk"], case["S"], case["page"]
    group, scale = case["Hq"] // Hk, 1.0 / math.sqrt(D)
    o = torch.zeros((B, case["Hq"], S, D), dtype=torch.float64, device="cuda")
    weight = st["weight"].double() if case["weights"] else None
    for b in range(B):
        n = int(st["lengths"][b])
        pages = st["pages"][b, : -(-n // P)].long()
        for h in range(Hk):
            k, v = _exact_rows(st["kv"][pages, h].reshape(-1, D * 5 // 4)[:n], D, dtype)
            total = torch.zeros(n, dtype=torch.float64, device="cuda")
            for i in range(S):
                see = n - S + i + 1
                p = torch.softmax(st["q"][b, h * group:(h + 1) * group, i].double() @ k[:see].T * scale, -1)
                o[b, h * group:(h + 1) * group, i] = p @ v[:see]
                total[:see] += p.sum(0)
            if weight is not None:
                slot = torch.arange(n, device="cuda")
                weight[pages[slot // P], h, slot % P] += total
    return o if weight is None else (o, weight)
