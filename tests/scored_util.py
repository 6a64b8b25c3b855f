"""Caches, rows and 64-bit oracles for the tests of scored paged attention, tracked writes and eviction: everything from the definitions, a sequence and head at a time."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}         # half a step, relative


def make_cache(L, nkv, hd, page, dtype, int8, g, dev, spare=2, fill=float("nan")):
    """Sequences of L[b] tokens in scattered pages -> (kv, scale, block_table, [K, V fp64 per sequence: [nkv, L, hd]]).  What no token occupies holds `fill` (8 bits: any byte, and NaN scales)."""
    B, M = len(L), -(-max(max(L), 1) // page) + 1
    nblk = B * M + spare
    bt = torch.randperm(nblk, generator=torch.Generator().manual_seed(11))[: B * M].reshape(B, M).int().to(dev)
    if int8:
        kv = torch.randint(-128, 128, (nblk, 2, nkv, page, hd), generator=g, device=dev, dtype=torch.int8)
        sc = torch.full((nblk, 2, nkv, page), float("nan"), device=dev)
    else:
        kv, sc = torch.full((nblk, 2, nkv, page, hd), fill, device=dev, dtype=dtype), None
    dense = []
    for b in range(B):
        k = torch.randn(nkv, L[b], hd, device=dev, generator=g)
        v = torch.randn(nkv, L[b], hd, device=dev, generator=g) + 0.5
        if int8:
            ks, vs = (x.abs().amax(-1, keepdim=True).clamp_min(1e-3) / 127 for x in (k, v))
            kc, vc = ((x / s).round().clamp(-128, 127) for x, s in ((k, ks), (v, vs)))
            k, v = kc.double() * ks.double(), vc.double() * vs.double()
            kw, vw = ((c.to(torch.int16) ^ 0x80).to(torch.uint8).view(torch.int8) for c in (kc, vc))
        else:
            kw, vw = k.to(dtype), v.to(dtype)
            k, v = kw.double(), vw.double()
        for t0 in range(0, L[b], page):
            c, blk = min(page, L[b] - t0), int(bt[b, t0 // page])
            kv[blk, 0, :, :c] = kw[:, t0:t0 + c]
            kv[blk, 1].view(nkv, hd, page)[:, :, :c] = vw[:, t0:t0 + c].transpose(1, 2)
            if int8:
                sc[blk, 0, :, :c], sc[blk, 1, :, :c] = ks[:, t0:t0 + c, 0], vs[:, t0:t0 + c, 0]
        dense.append((k, v))
    return kv, sc, bt, dense


def gather_plane(plane, bt, b, n):
    """[nkv, n] of a plane for the first n slots of a sequence."""
    return plane[bt[b].long()].transpose(0, 1).reshape(plane.shape[1], -1)[:, :n]


def attend(q, k, v, lo, hi, *, scale, cap=0.0, slopes=None, positions=None, key_pos=None):
    """One sequence: q [n, nh, hd] (16 bit), k, v [nkv, L, hd] fp64, lo, hi [n] -> out, lse, weights [nkv, L] and the bounds' parts: sum p |v|, the size of a score's terms."""
    n, nh, hd = q.shape
    nkv, L = k.shape[0], k.shape[1]
    G, dev = nh // nkv, q.device
    out, pv = torch.zeros(2, n, nh, hd, dtype=torch.float64, device=dev)
    lse = torch.full((n, nh), float("-inf"), dtype=torch.float64, device=dev)
    size = torch.zeros(n, nh, dtype=torch.float64, device=dev)
    w = torch.zeros(nkv, L, dtype=torch.float64, device=dev)
    slot = torch.arange(L, device=dev)
    seen = (slot[None] >= lo[:, None]) & (slot[None] < hi[:, None])
    some = seen.any(1)
    for h in range(nh):
        kh = h // G
        u = q[:, h].double() @ k[kh].t().contiguous() * scale
        size[:, h] = (q[:, h].double().abs() @ k[kh].abs().t().contiguous() * abs(scale)).masked_fill(~seen, 0).amax(1) if L else 0
        s = cap * torch.tanh(u / cap) if cap else u
        if slopes is not None:
            kp = slot if key_pos is None else key_pos[kh]
            bias = slopes[h].double() * (kp[None] - positions[:, None]).double()
            size[:, h] += bias.abs().masked_fill(~seen, 0).amax(1)
            s = s + bias
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        lse[:, h] = torch.where(some, torch.logsumexp(s, -1), lse[:, h])
        out[:, h], pv[:, h] = p @ v[kh], p @ v[kh].abs()
        w[kh] += p.sum(0)
    return out, lse, w, pv, size


def bounds(dtype, hd, L, pv, size, out):
    """Errors allowed in (out, lse, a probability, relative).  A score is hd products summed in fp32 (hd 2^-24 of the sum of their sizes), scaled, capped and biased (16 more roundings of that
    size): eps.  exp gives its share 2 eps (weight and sum) and 2^-22 for itself; the running maximum rescales every 32 keys at most (2^-24 each).  The probabilities are rounded to the
    activation's type before the second product, and the result once more."""
    eps = (hd + 16) * 2.0 ** -24 * size
    rel = 2 * eps + 2.0 ** -21 + (L / 32 + 8) * 2.0 ** -24
    u = U[dtype]
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0            # fp16 has no numbers below its smallest: a step of probabilities and results
    return u * (out.abs() + pv) + rel[..., None] * 2 * pv + tiny * (1 + L ** 0.5), eps + rel, rel


def evict(w, pos, n, keep, newest, sinks, recent, bad=None):
    """One (sequence, head): lists of weights and positions -> [(source, hole)] as the definition has them."""
    if n <= keep:
        return []
    def rank(t):
        if bad is not None and bad(t):
            return (0, 0.0)
        if pos[t] < sinks or pos[t] >= newest - recent:
            return (3, 0.0)
        return (0, 0.0) if math.isnan(w[t]) else (1, w[t] + 0.0)
    order = sorted(range(n), key=lambda t: (tuple(-x for x in rank(t)), t))
    kept = set(order[:keep])
    return list(zip([t for t in range(keep, n) if t in kept], [t for t in range(keep) if t not in kept]))
