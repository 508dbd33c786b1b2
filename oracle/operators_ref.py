"""Plain restatements in 64 bits of the operators around attention: rotary positions, the 4-bit cache, attention
over it and eviction from it.  Test infrastructure only; works on CPU and CUDA tensors, one row at a time where that
is the clearest.  The reference project has none of these operators: what is restated are their formulas.
"""
import math

import torch


# ------------------------------------------------------------------ rotary positions

def frequencies(dim, base=10000.0, scaling="none", factor=1.0, original_length=0, turns=None):
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    out = []
    low, high = turns or {"yarn": (1.0, 32.0), "bands": (1.0, 4.0)}.get(scaling, (0.0, 0.0))
    if scaling == "yarn":
        pair = lambda t: dim * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), dim - 1)
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        if scaling == "linear" or (scaling == "ntk" and dim == 2):
            f /= factor
        elif scaling == "yarn":
            ramp = min(max((i - first) / max(last - first, 0.001), 0.0), 1.0)
            f = f * (1 - ramp) + f / factor * ramp
        elif scaling == "bands":
            share = min(max((original_length * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f * share + f / factor * (1 - share)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def rotary_table(length, dim, multiplier=1.0, **scaling):
    angle = torch.arange(length, dtype=torch.float64)[:, None] * frequencies(dim, **scaling)
    return torch.stack((angle.cos(), angle.sin()), -1) * multiplier


def rotary(x, table, positions=None, interleaved=False, inverse=False):
    """x [B, H, S, D] in 64 bits, turned by table [length, dim / 2, 2] (any float type)."""
    B, H, S, D = x.shape
    n = table.shape[1]
    pos = torch.arange(S, device=x.device) if positions is None else positions.long()
    cs = table.double()[pos.expand(B, S)][:, None]
    c, s = cs[..., 0], cs[..., 1] * (-1 if inverse else 1)
    y = x.double().clone()
    first = torch.arange(n, device=x.device) * 2 if interleaved else torch.arange(n, device=x.device)
    second = first + (1 if interleaved else n)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


# ------------------------------------------------------------------ the record

def code_places(D):
    """(byte, bit) of every dim's K code and V code in a record of 5 D / 4 bytes."""
    G, k, v = D // 32, [], []
    for d in range(D):
        w, r = d // 32, d % 32
        c, j = r // 8, r % 8
        k.append(((w // 4) * 64 + c * 4 * min(G, 4) + 4 * (w % 4) + j // 2, 4 * (j % 2)))
        g, i = r // 4, r % 4
        v.append((D // 2 + g * (D // 16) + 2 * w + i // 2, 4 * (i % 2)))
    return k, v


def quantise(x):
    """16-bit rows [n, D] -> (codes [n, D], scale [n, G], minimum [n, G]), in the operator's own 32-bit steps."""
    f = x.float().reshape(x.shape[0], x.shape[1] // 32, 32)
    lo, hi = f.min(-1).values, f.max(-1).values
    rng = hi - lo
    scale = (rng * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).to(x.dtype)
    scale = torch.where(scale.float() < 2.0 ** -126, torch.zeros_like(scale), scale)
    inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(rng))
    u = ((f - lo[..., None]) * inv[..., None]).round().clamp(0, 15)
    bad = ~(rng < math.inf)
    u = torch.where(bad[..., None], torch.zeros_like(u), u)
    nan = torch.full_like(scale, math.nan)
    return u.reshape(x.shape).to(torch.int64), torch.where(bad, nan, scale), torch.where(bad, nan, lo.to(x.dtype))


def records(k, v):
    """K and V rows [n, D] -> records [n, 5 D / 4]."""
    n, D = k.shape
    out = torch.zeros((n, 5 * D // 4), dtype=torch.uint8, device=k.device)
    at = D
    for x, places in zip((k, v), code_places(D)):
        u, scale, lo = quantise(x)
        for d, (byte, bit) in enumerate(places):
            out[:, byte] |= (u[:, d] << bit).to(torch.uint8)
        pairs = torch.stack((scale, lo), -1).reshape(n, 2 * scale.shape[1]).contiguous().view(torch.uint8)
        out[:, at:at + pairs.shape[1]] = pairs
        at += pairs.shape[1]
    return out


def values(rec, dtype):
    """Records [n, 5 D / 4] -> (K values, V values, V values less those of code 8) in 64 bits."""
    n, D = rec.shape[0], rec.shape[1] * 4 // 5
    G, out, at = D // 32, [], D
    for places in code_places(D):
        u = torch.stack([(rec[:, byte] >> bit) & 15 for byte, bit in places], -1).double()
        pairs = rec[:, at:at + 4 * G].contiguous().view(dtype).double().reshape(n, G, 2)
        at += 4 * G
        scale = pairs[..., 0].repeat_interleave(32, -1)
        out.append(u * scale + pairs[..., 1].repeat_interleave(32, -1))
    return out[0], out[1], (u - 8) * scale


def rows_of(kv, table, b, h, n):
    """The first n records of head h of sequence b."""
    P = kv.shape[2]
    slot = torch.arange(n, device=kv.device)
    return kv[table[b].long()[slot // P], h, slot % P]


# ------------------------------------------------------------------ attention and eviction

def attention(q, kv, table, lengths, sm_scale, counts=None):
    """(o, lse, weights {(b, h): [n]}, bound) in 64 bits; bound: per output, the sums its error is made of
    (sum p s |u - 8|, sum p |m + 8 s|, sum p (|m| + 8 s), sum p |v|, largest sum |q| |k| of a visible token)."""
    B, Hq, S, D = q.shape
    H, dev = kv.shape[1], q.device
    o = torch.zeros((B, Hq, S, D), dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=dev)
    parts, middles, both, sizes = (torch.zeros_like(o) for _ in range(4))
    terms = torch.zeros_like(lse)
    weights = {}
    for b in range(B):
        n = int(lengths[b])
        count = S if counts is None else min(int(counts[b]), S)
        for h in range(H):
            rec = rows_of(kv, table, b, h, n)
            k, v, part = values(rec, q.dtype)
            eight = rec[:, -(D // 8):].contiguous().view(q.dtype)[:, ::2].double().repeat_interleave(32, -1) * 8     # 8 s of V
            apart = (v - part - eight).abs() + eight
            total = torch.zeros(n, dtype=torch.float64, device=dev)
            for hq in range(h * (Hq // H), (h + 1) * (Hq // H)):
                for i in range(count):
                    see = n - count + i + 1
                    if see <= 0:
                        continue
                    x = q[b, hq, i].double()
                    s = k[:see] @ x * sm_scale
                    lse[b, hq, i] = torch.logsumexp(s, 0)
                    p = torch.exp(s - lse[b, hq, i])
                    o[b, hq, i], parts[b, hq, i], middles[b, hq, i] = p @ v[:see], p @ part[:see].abs(), p @ (v - part)[:see].abs()
                    sizes[b, hq, i], both[b, hq, i] = p @ v[:see].abs(), p @ apart[:see]
                    terms[b, hq, i] = (k[:see].abs() @ x.abs()).max() * abs(sm_scale)
                    total[:see] += p
            weights[b, h] = total
    return o, lse, weights, (parts, middles, both, sizes, terms)


def evict(weight, position, budget, recent):
    """Which of n slots a head keeps and what moves: ([(to, from)], kept slots) for weight [n] and position [n]."""
    n = weight.shape[0]
    if n <= budget:
        return [], list(range(n))
    w, pos = weight.tolist(), position.tolist()
    newest = max(pos)
    def key(s):
        if pos[s] > newest - recent:
            return (0, 0.0, s)
        return (1, -w[s] if w[s] > 0 else 0.0, s)
    kept = sorted(sorted(range(n), key=key)[:budget])
    holes = [s for s in range(budget) if s not in set(kept)]
    movers = [s for s in kept if s >= budget]
    return list(zip(holes, movers)), kept
