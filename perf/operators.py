"""What the speed of the scored paged attention and of the cache that forgets is measured on: single calls of

  attend  ``ops.paged_attention_scored``: decode rows and chunks of rows over a paged cache, scores capped by a tanh or biased by distance, rows that
          see an interval of the cache (causal, a window, a prefix that all rows see, documents), log-sum-exps, and the attention weight that each cached
          token has drawn so far;
  write   ``ops.rope_kv_write_slots``: new rows into slots of their own, rotated at their positions;
  evict   ``ops.kv_evict``: a cache brought back to its budget by accumulated attention weight.

Caches, rows and weights are random, made on the device from the seed.  Keys and queries are scaled so that a row's weight lies on a few dozen tokens,
values have a mean per channel, and slots behind a sequence's length hold what an earlier sequence left there.  Heads and pages are those of the models that the other
benchmark runs (28 over 4 heads of 128, 14 over 2 of 64), of a tensor-parallel shard (8 over 1) and of 32 over 8."""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SINKS, RECENT = 4, 32       # tokens that no eviction takes: the first and the newest


def listed():
    return [
        # one user: launches and latency
        dict(name="attend-b1", kind="attend", batch=1, rows=1, ctx=1000, ragged=False, nh=28, nkv=4, hd=128, page=16, dtype="fp16", kv="16", mask="causal", cap=50.0, alibi=False, track=False, evicted=False),
        # a full batch of a model with distance biases
        dict(name="attend-b64-bias", kind="attend", batch=64, rows=1, ctx=1024, ragged=True, nh=28, nkv=4, hd=128, page=16, dtype="bf16", kv="16", mask="causal", cap=0.0, alibi=True, track=False, evicted=False),
        # an odd batch over an 8-bit cache with large pages, weights kept for eviction
        dict(name="attend-b13-int8-track", kind="attend", batch=13, rows=1, ctx=4096, ragged=True, nh=32, nkv=8, hd=128, page=64, dtype="fp16", kv="int8", mask="causal", cap=30.0, alibi=False, track=True, evicted=False),
        # a shard's long contexts after evictions: positions are not slots
        dict(name="attend-b4-32k-evicted", kind="attend", batch=4, rows=1, ctx=32000, ragged=False, nh=8, nkv=1, hd=128, page=16, dtype="bf16", kv="16", mask="causal", cap=0.0, alibi=True, track=True, evicted=True),
        # a batch of prompts under capped scores
        dict(name="attend-8x512-cap", kind="attend", batch=8, rows=512, ctx=0, ragged=False, nh=28, nkv=4, hd=128, page=16, dtype="fp16", kv="16", mask="causal", cap=50.0, alibi=False, track=False, evicted=False),
        # packed documents in small heads, prompts of unequal, odd length
        dict(name="attend-docs-3x1501", kind="attend", batch=3, rows=1501, ctx=0, ragged=True, nh=14, nkv=2, hd=64, page=32, dtype="bf16", kv="16", mask="documents", cap=0.0, alibi=False, track=False, evicted=False),
        # a prefix that all rows see, an odd chunk behind cached tokens, 8-bit cache, distance biases
        dict(name="attend-prefix-333-int8", kind="attend", batch=1, rows=333, ctx=3001, ragged=False, nh=28, nkv=4, hd=128, page=16, dtype="fp16", kv="int8", mask="prefix", cap=0.0, alibi=True, track=False, evicted=False),
        # long prompts in portions, weights kept for eviction
        dict(name="attend-2x2048-track", kind="attend", batch=2, rows=2048, ctx=2048, ragged=False, nh=28, nkv=4, hd=128, page=16, dtype="fp16", kv="16", mask="causal", cap=0.0, alibi=False, track=True, evicted=False),
        # a decode step's rows into a cache after evictions
        dict(name="write-b64", kind="write", batch=64, rows=1, ctx=1024, nh=28, nkv=4, hd=128, page=16, dtype="fp16"),
        # prompts' rows
        dict(name="write-8x512", kind="write", batch=8, rows=512, ctx=0, nh=28, nkv=4, hd=128, page=16, dtype="bf16"),
        # one user's cache brought back to its budget after a few hundred tokens
        dict(name="evict-b1", kind="evict", batch=1, length=2304, keep=2048, ragged=False, nkv=4, hd=128, page=16, dtype="fp16"),
        # a full batch of prompts cut to a quarter
        dict(name="evict-b64", kind="evict", batch=64, length=4096, keep=1024, ragged=True, nkv=4, hd=128, page=16, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["attend", "write", "evict"], [7, 2, 3])[0]
    nh, nkv, hd = rng.choice([(28, 4, 128), (14, 2, 64), (8, 1, 128), (32, 8, 128)])
    common = dict(nkv=nkv, hd=hd, page=rng.choice([16, 16, 32, 64]), dtype=rng.choice(["fp16", "bf16"]))
    if kind == "write":
        rows = rng.choice([1, 1, _log(rng, 2, 512)])
        return dict(kind=kind, batch=_log(rng, 1, max(1, min(64, 4096 // rows))), rows=rows, ctx=_log(rng, 1, 2048), nh=nh, **common)
    if kind == "evict":
        length = _log(rng, 128, 4096)
        return dict(kind=kind, batch=_log(rng, 1, 64), length=length, keep=max(SINKS + RECENT, int(length * rng.uniform(0.2, 0.95))), ragged=rng.random() < 0.5, **common)
    kv = rng.choice(["16", "16", "int8"])
    cap = rng.choice([0.0, 30.0, 50.0])
    alibi = rng.random() < 0.4
    if rng.random() < 0.5:                                             # decode
        ctx = _log(rng, 64, 32768)
        evicted = rng.random() < 0.3
        return dict(kind=kind, batch=_log(rng, 1, max(1, min(64, 131072 // ctx))), rows=rng.choice([1, 1, 1, 2, 4]), ctx=ctx, ragged=rng.random() < 0.6, nh=nh, kv=kv,
                    mask="causal" if evicted else rng.choice(["causal", "causal", "window"]), cap=cap, alibi=alibi, track=rng.random() < 0.5, evicted=evicted, **common)
    rows = _log(rng, 16, 2048)
    ctx = rng.choice([0, _log(rng, 16, 2048)])
    return dict(kind=kind, batch=_log(rng, 1, max(1, min(8, 4096 // rows))), rows=rows, ctx=ctx, ragged=rng.random() < 0.5, nh=nh, kv=kv,
                mask=rng.choice(["causal", "causal", "prefix", "documents", "window"]), cap=cap, alibi=alibi, track=rng.random() < 0.3, evicted=False, **common)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _shape(c):
    """Host numbers of a case, the same for every seed: (rows of each sequence, cached tokens in front of them)."""
    n, r = c["batch"], c.get("rows", 1)
    if not c.get("ragged"):
        return [r] * n, [c["ctx"]] * n
    part = [(((b * 7 + 3) % 13) / 13 + 0.3) / 1.3 for b in range(n)]
    part[n // 2] = 1.0
    return [max(1, int(r * p)) if r > 1 else 1 for p in part], [max(0, int(c["ctx"] * p)) for p in part]


def _intervals(c, b, rows, ctx, seed):
    """(begin, end) of a sequence's rows: host lists of slots."""
    pos = range(ctx, ctx + rows)
    end = [p + 1 for p in pos]
    if c["mask"] == "window":
        return [max(0, p + 1 - max(8, (ctx + rows) // 3)) for p in pos], end
    if c["mask"] == "prefix":
        prefix = ctx + rows // 4
        return [0] * rows, [max(e, prefix) for e in end]
    if c["mask"] == "documents":
        step = max(1, (ctx + rows) // 5 + (seed + b) % 7)
        return [p // step * step for p in pos], end
    return [0] * rows, end


def _pages(blocks, per, gen):
    return torch.randperm(blocks * per, generator=gen, device=DEV).reshape(blocks, per).int()


def _cache(nblk, c, gen):
    """A pool with keys token by token and values channel by channel, as the framework's writer leaves them; 8 bits: the byte is code + 128."""
    nkv, hd, page, dt = c["nkv"], c["hd"], c["page"], DTYPES[c["dtype"]]
    k = torch.randn(nblk, nkv, page, hd, device=DEV, generator=gen)
    v = torch.randn(nblk, nkv, hd, page, device=DEV, generator=gen) + torch.randn(nkv, hd, 1, device=DEV, generator=gen) * 0.5
    kv = torch.empty(nblk, 2, nkv, page, hd, device=DEV, dtype=torch.int8 if c.get("kv") == "int8" else dt)
    if c.get("kv") != "int8":
        kv[:, 0], kv[:, 1] = k, v.view(nblk, nkv, page, hd)
        return kv, None
    scale = torch.stack([k.abs().amax(-1), v.abs().amax(-2)], 1) / 127                       # [nblk, 2, nkv, page]
    code = lambda x, s: ((x / s).round().clamp(-128, 127).to(torch.int16) ^ 0x80).to(torch.uint8).view(torch.int8)
    kv[:, 0] = code(k, scale[:, 0].unsqueeze(-1))
    kv[:, 1] = code(v, scale[:, 1].unsqueeze(-2)).view(nblk, nkv, page, hd)
    return kv, scale.contiguous()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    nkv, hd, page, dt, B = c["nkv"], c["hd"], c["page"], DTYPES[c["dtype"]], c["batch"]
    s = dict(case=c, kind=c["kind"], nkv=nkv, hd=hd, page=page)
    if c["kind"] == "evict":
        keep = c["keep"]
        lens = [c["length"] if not c["ragged"] else max(1, int(c["length"] * (((b * 5 + 2) % 11) / 11 + 0.4) / 1.4)) for b in range(B)]
        lens[B // 2] = c["length"]
        M = -(-c["length"] // page)
        s["block_table"] = _pages(B, M, gen)
        s["kv"], _ = _cache(B * M, c, gen)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["next_pos"] = s["lens"] + 100                                                       # 100 tokens are gone already
        # positions: those left by an earlier eviction in any order, then the tokens since; weights: a few tokens drew most of the attention
        at = torch.arange(M * page, device=DEV).expand(B, nkv, -1)
        old = torch.rand(B, nkv, M * page, device=DEV, generator=gen)
        shuffled = torch.where(at < keep // 2, old, 2 + at / (M * page)).argsort(-1)
        pos = torch.where(shuffled < SINKS, shuffled, shuffled + 100).int()
        w = torch.exp(torch.randn(B, nkv, M * page, device=DEV, generator=gen) * 2 - 4)
        both = torch.zeros(2, B * M, nkv, page, dtype=torch.int32, device=DEV)                # the two planes behind each other, so that one copy restores them
        place = s["block_table"].long().reshape(-1)
        both[0, place] = w.view(torch.int32).reshape(B, nkv, M, page).transpose(1, 2).reshape(B * M, nkv, page)
        both[1, place] = pos.reshape(B, nkv, M, page).transpose(1, 2).reshape(B * M, nkv, page)
        s["planes"], s["planes_saved"] = both, both.clone()
        s["weights"], s["key_pos"] = both[0].view(torch.float32), both[1]
        return s
    rows, ctx = _shape(c)
    L = max(r + x for r, x in zip(rows, ctx))
    M = -(-L // page)
    s["block_table"] = _pages(B, M, gen)
    s["kv"], s["scale"] = _cache(B * M, c, gen)
    T, nh = sum(rows), c["nh"]
    s.update(nh=nh, max_len=M * page, q_len=max(rows), rows=T)
    s["row_start"] = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    s["row_seq"] = torch.repeat_interleave(torch.arange(B, dtype=torch.int32, device=DEV), torch.tensor(rows, device=DEV))
    slots = torch.tensor([x + i for r, x in zip(rows, ctx) for i in range(r)], dtype=torch.int32, device=DEV)
    if c["kind"] == "write":
        s["slots"], s["positions"] = slots, slots + 137
        s["qkv"] = torch.randn(T, (nh + 2 * nkv) * hd, device=DEV, generator=gen).to(dt)
        s["bias"] = (torch.randn((nh + 2 * nkv) * hd, device=DEV, generator=gen) * 0.1).to(dt)
        ang = torch.arange(L + 137, dtype=torch.float64, device=DEV)[:, None] * 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) / (hd // 2))
        s["cos_sin"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s["weights"] = torch.rand(B * M, nkv, page, device=DEV, generator=gen)
        s["key_pos"] = torch.zeros(B * M, nkv, page, dtype=torch.int32, device=DEV)
        return s
    s["q"] = (torch.randn(T, nh, hd, device=DEV, generator=gen) * 3).to(dt)
    spans = [_intervals(c, b, r, x, seed) for b, (r, x) in enumerate(zip(rows, ctx))]
    begin, end = ([v for sp in spans for v in sp[i]] for i in (0, 1))
    s["begin"] = torch.tensor(begin, dtype=torch.int32, device=DEV) if c["mask"] in ("window", "documents") else None
    s["end"] = torch.tensor(end, dtype=torch.int32, device=DEV)
    s["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], device=DEV) if c["alibi"] else None
    s["positions"] = slots + (L if c["evicted"] else 0) if c["alibi"] else None
    s["key_pos"] = None
    if c["evicted"] and c["alibi"]:
        old = torch.rand(B * M, nkv, page, device=DEV, generator=gen)
        s["key_pos"] = (old * (2 * L)).int() % max(1, L)
    s["weights"] = torch.rand(B * M, nkv, page, device=DEV, generator=gen) if c["track"] else None
    s["decay"] = 0.9 if c["evicted"] else 1.0
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["kind"] == "attend":
        return _attend_own(s) if own else _attend_plain(s)
    if s["kind"] == "write":
        return _write_own(s) if own else _write_plain(s)
    s["planes"].copy_(s["planes_saved"])             # what the steps since the last eviction have left
    return _evict_own(s) if own else _evict_plain(s)


def _attend_own(s):
    from rtp_llm_amd import ops
    out, lse = ops.paged_attention_scored(s["q"], s["kv"], s["scale"], s["block_table"], s["end"], s["nkv"], s["page"], s["max_len"], begin=s["begin"],
                                          row_start=s["row_start"], q_len=s["q_len"], softcap=s["case"]["cap"], slopes=s["slopes"], positions=s["positions"],
                                          key_pos=s["key_pos"], weights=s["weights"], decay=s["decay"], return_lse=True)
    return {"out": out, "lse": lse, **({"weights": s["weights"]} if s["weights"] is not None else {})}


def _write_own(s):
    from rtp_llm_amd import ops
    q = ops.rope_kv_write_slots(s["qkv"], s["bias"], s["cos_sin"], s["positions"], s["slots"], s["block_table"], s["kv"], None, s["nh"], s["nkv"], s["hd"], s["page"],
                                row_seq=s["row_seq"], key_pos=s["key_pos"], weights=s["weights"])
    return {"q": q, "kv": s["kv"], "key_pos": s["key_pos"], "weights": s["weights"]}


def _evict_own(s):
    from rtp_llm_amd import ops
    lens = ops.kv_evict(s["weights"], s["key_pos"], s["block_table"], s["lens"], s["next_pos"], s["kv"], None, s["case"]["keep"], sinks=SINKS, recent=RECENT)
    return {"lens": lens, "kv": s["kv"], "key_pos": s["key_pos"], "weights": s["weights"]}


def _dense(s):
    """Keys and values of every sequence, fp32 [B, nkv, slots, hd]."""
    t, nkv, hd, page = s["block_table"].long(), s["nkv"], s["hd"], s["page"]
    B, M = t.shape
    got = s["kv"][t]                                                                          # [B, M, 2, nkv, page, hd]
    x = got.float() if s["scale"] is None else (got.view(torch.uint8).float() - 128)
    k, v = x[:, :, 0], x[:, :, 1].reshape(B, M, nkv, hd, page).transpose(-1, -2)
    if s["scale"] is not None:
        sc = s["scale"][t]
        k, v = k * sc[:, :, 0].unsqueeze(-1), v * sc[:, :, 1].unsqueeze(-1)
    return tuple(y.transpose(1, 2).reshape(B, nkv, M * page, hd) for y in (k, v))


def _attend_plain(s):
    c, nkv, nh, hd, n = s["case"], s["nkv"], s["nh"], s["hd"], s["q_len"]
    B, L, G, dev = s["block_table"].shape[0], s["max_len"], s["nh"] // s["nkv"], s["q"].device
    k, v = _dense(s)
    place = s["row_start"][:-1, None].long() + torch.arange(n, device=dev)                   # [B, n]: a sequence's rows, the last ones of short sequences not its own
    mine = place < s["row_start"][1:, None]
    place = torch.where(mine, place, 0)
    q = s["q"][place].float().reshape(B, n, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, n * G, hd)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(hd)).view(B, nkv, n, G, L)
    if c["cap"] > 0:
        x = x.div_(c["cap"]).tanh_().mul_(c["cap"])
    slot = torch.arange(L, device=dev)
    if s["slopes"] is not None:
        kp = slot.expand(B, nkv, L) if s["key_pos"] is None else s["key_pos"][s["block_table"].long()].transpose(1, 2).reshape(B, nkv, L)
        far = kp[:, :, None, :] - s["positions"][place][:, None, :, None]                   # [B, nkv, n, L]
        x = x.add_(s["slopes"].view(1, nkv, 1, G, 1) * far.unsqueeze(3))
    seen = (slot < s["end"][place].unsqueeze(-1)) & mine.unsqueeze(-1)
    if s["begin"] is not None:
        seen &= slot >= s["begin"][place].unsqueeze(-1)
    x = x.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp_min_(-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    p = p.div_(total.clamp_min(1e-30))
    out = torch.matmul(p.view(B, nkv, n * G, L), v).view(B, nkv, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B, n, nh * hd)
    ans = {"out": out[mine].to(s["q"].dtype), "lse": lse.permute(0, 2, 1, 3).reshape(B, n, nh)[mine]}
    if s["weights"] is not None:
        w = s["weights"]
        gain = p.sum((2, 3)).view(B, nkv, -1, s["page"]).transpose(1, 2)                     # [B, M, nkv, page]
        reach = torch.where(mine, s["end"][place], 0).amax(1)
        old = w[s["block_table"].long()]
        used = (slot < reach[:, None]).view(B, -1, 1, s["page"])
        w[s["block_table"].long()] = torch.where(used, old * s["decay"] + gain, old)
        ans["weights"] = w
    return ans


def _write_plain(s):
    nh, nkv, hd, page, dt = s["nh"], s["nkv"], s["hd"], s["page"], s["qkv"].dtype
    x = (s["qkv"].float() + s["bias"].float()).to(dt).float().view(s["rows"], nh + 2 * nkv, hd)  # the linear's output is a 16-bit tensor
    cs = s["cos_sin"][s["positions"].long()]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    turned = torch.cat([cos * a - sin * b, cos * b + sin * a], -1).to(dt)
    blk, tok = s["block_table"][s["row_seq"].long(), s["slots"].long() // page].long(), s["slots"].long() % page
    s["kv"][:, 0][blk, :, tok] = turned[:, nh: nh + nkv]
    s["kv"][:, 1].view(-1, nkv, hd, page)[blk, :, :, tok] = x[:, nh + nkv:].to(dt)
    s["key_pos"][blk, :, tok] = s["positions"][:, None].expand(-1, nkv)
    s["weights"][blk, :, tok] = 0
    return {"q": turned[:, :nh].contiguous(), "kv": s["kv"], "key_pos": s["key_pos"], "weights": s["weights"]}


def _evict_plain(s):
    keep, nkv, hd, page, t = s["case"]["keep"], s["nkv"], s["hd"], s["page"], s["block_table"].long()
    B, M = t.shape
    L = M * page
    flat = lambda x: x[t].transpose(1, 2).reshape(B, nkv, L)
    w, pos, slot, n = flat(s["weights"]), flat(s["key_pos"]), torch.arange(L, device=t.device), s["lens"].view(B, 1, 1)
    safe = (pos < SINKS) | (pos >= s["next_pos"].view(B, 1, 1) - RECENT)
    w = w.masked_fill(safe, float("inf")).masked_fill(slot >= n, float("-inf"))
    order = w.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(B, nkv, L, dtype=torch.bool, device=t.device).scatter_(-1, order[..., :keep], True) & (slot < n)
    hole = ~kept & (slot < keep) & (slot < n)
    late = kept & (slot >= keep)
    hb, hh, to = hole.nonzero(as_tuple=True)                                                 # in the order of sequence, head, slot: the i-th hole takes the i-th late token
    _, _, frm = late.nonzero(as_tuple=True)
    b0, t0, b1, t1 = t[hb, to // page], to % page, t[hb, frm // page], frm % page
    s["kv"][:, 0][b0, hh, t0] = s["kv"][:, 0][b1, hh, t1]
    v = s["kv"][:, 1].view(-1, nkv, hd, page)
    v[b0, hh, :, t0] = v[b1, hh, :, t1]
    for x in (s["weights"], s["key_pos"]):
        x[b0, hh, t0] = x[b1, hh, t1]
    return {"lens": s["lens"].clamp(max=keep), "kv": s["kv"], "key_pos": s["key_pos"], "weights": s["weights"]}


# ---------------------------------------------------------------------------------------------------------------- costs
def work(case):
    c = case
    es = 1 if c.get("kv") == "int8" else 2
    token = c["nkv"] * (2 * c["hd"] * es + (8 if c.get("kv") == "int8" else 0))               # a cached token: keys, values, scales
    if c["kind"] == "evict":
        lens = [c["length"] if not c["ragged"] or b == c["batch"] // 2 else max(1, int(c["length"] * (((b * 5 + 2) % 11) / 11 + 0.4) / 1.4)) for b in range(c["batch"])]
        moved = sum(max(0, n - c["keep"]) * c["keep"] / n for n in lens)                      # of tokens whose weight does not depend on their slot
        return {"bytes": sum(lens) * c["nkv"] * 8 + moved * 2 * (token + 8 * c["nkv"]), "flops": 0.0}
    rows, ctx = _shape(c)
    T, width = sum(rows), c["nh"] * c["hd"]
    if c["kind"] == "write":
        return {"bytes": T * ((width + 2 * c["nkv"] * c["hd"]) * 4 + 8 * c["nkv"]), "flops": T * 6.0 * (c["nh"] + c["nkv"]) * c["hd"]}
    seen = reach = 0
    for b, (r, x) in enumerate(zip(rows, ctx)):
        lo, hi = _intervals(c, b, r, x, 0)
        seen += sum(hi) - sum(lo)
        reach += max(hi) - min(lo)
    return {"bytes": reach * (token + (8 * c["nkv"] if c["track"] else 0) + (4 * c["nkv"] if c["evicted"] and c["alibi"] else 0)) + T * (4 * width + 4 * c["nh"]),
            "flops": 4.0 * c["hd"] * c["nh"] * seen}


# ---------------------------------------------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "write": _write_exact, "evict": _evict_exact}[s["kind"]](s)


def _attend_exact(s):
    """Row by row of the definition, a key/value head of a sequence at a time."""
    c, hd, nkv, page = s["case"], s["hd"], s["nkv"], s["page"]
    G = s["nh"] // nkv
    out = torch.zeros(s["rows"], s["nh"], hd, dtype=torch.float64, device=DEV)
    lse = torch.full((s["rows"], s["nh"]), float("-inf"), dtype=torch.float64, device=DEV)
    w = None if s["weights"] is None else s["weights"].double()
    start = s["row_start"].tolist()
    for b in range(len(start) - 1):
        r0, r1 = start[b], start[b + 1]
        hi = s["end"][r0:r1].long()
        lo = torch.zeros_like(hi) if s["begin"] is None else s["begin"][r0:r1].long()
        L = int(hi.max())
        pages = s["block_table"][b, : -(-L // page)].long()
        slot = torch.arange(L, device=DEV)
        hidden = (slot[None] < lo[:, None]) | (slot[None] >= hi[:, None])
        for h in range(nkv):
            k = s["kv"][pages, 0, h].reshape(-1, hd)[:L]
            v = s["kv"][pages, 1, h].reshape(-1, hd, page).permute(0, 2, 1).reshape(-1, hd)[:L]
            if s["scale"] is not None:
                ks, vs = (s["scale"][pages, i, h].reshape(-1)[:L, None].double() for i in (0, 1))
                k, v = (k.to(torch.int64) & 255).double().sub(128) * ks, (v.to(torch.int64) & 255).double().sub(128) * vs
            k, v = k.double(), v.double()
            for g in range(h * G, h * G + G):
                a = s["q"][r0:r1, g].double() @ k.t().contiguous() / hd ** 0.5
                if c["cap"]:
                    a = c["cap"] * torch.tanh(a / c["cap"])
                if s["slopes"] is not None:
                    kp = slot if s["key_pos"] is None else s["key_pos"][pages, h].reshape(-1)[:L]
                    a = a + s["slopes"][g].double() * (kp[None] - s["positions"][r0:r1, None]).double()
                a[hidden] = float("-inf")
                lse[r0:r1, g] = torch.logsumexp(a, -1)
                p = torch.softmax(a, -1)
                out[r0:r1, g] = p @ v
                if w is not None:
                    if g == h * G:
                        old = w[pages, h].reshape(-1).clone()
                        old[:L] *= s["decay"]
                    old[:L] += p.sum(0)
            if w is not None:
                w[pages, h] = old.view(-1, page)
    return {"out": out.flatten(1), "lse": lse, **({"weights": w} if w is not None else {})}


def _write_exact(s):
    nh, nkv, hd, page, dt = s["nh"], s["nkv"], s["hd"], s["page"], s["qkv"].dtype
    x = (s["qkv"].double() + s["bias"].double()).to(dt).double().reshape(-1, nh + 2 * nkv, 2, hd // 2)
    angle = torch.view_as_complex(s["cos_sin"].double())[s["positions"].long()][:, None]
    z = torch.complex(x[:, : nh + nkv, 0], x[:, : nh + nkv, 1]) * angle
    turned = torch.cat([z.real, z.imag], -1)
    kv, pos, w = s["kv"].double(), s["key_pos"].clone(), s["weights"].double()
    seq, slot = s["row_seq"].long(), s["slots"].long()
    blk, tok = s["block_table"].long()[seq, torch.div(slot, page, rounding_mode="floor")], slot.remainder(page)
    head = torch.arange(nkv, device=DEV)[None]
    at, tk = blk[:, None], tok[:, None]
    kv[at, 0, head, tk] = turned[:, nh:]
    vv = kv[:, 1].reshape(-1, nkv, hd, page).permute(0, 1, 3, 2).contiguous()
    vv[at, head, tk] = x[:, nh + nkv:].flatten(2)
    kv[:, 1] = vv.permute(0, 1, 3, 2).reshape(-1, nkv, page, hd)
    pos[at, head, tk] = s["positions"][:, None]
    w[at, head, tk] = 0.0
    return {"q": turned[:, :nh], "kv": kv, "key_pos": pos, "weights": w}


def _evict_exact(s):
    """A sequence and head at a time: the kept slots by sorting pairs, then token for token."""
    keep, page, nkv, hd = s["case"]["keep"], s["page"], s["nkv"], s["hd"]
    kv, w, pos = s["kv"].clone(), s["weights"].clone(), s["key_pos"].clone()
    lens, nxt, tables = s["lens"].tolist(), s["next_pos"].tolist(), s["block_table"].long()
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        slots = torch.arange(n, device=DEV)
        blk, tok = tables[b, slots // page], slots % page
        for h in range(nkv):
            ww, pp = s["weights"][blk, h, tok].double(), s["key_pos"][blk, h, tok]
            ww[(pp < SINKS) | (pp >= nxt[b] - RECENT)] = float("inf")
            top = torch.sort(-ww, stable=True).indices[:keep].sort().values
            late = top[top >= keep]
            inside = torch.ones(keep, dtype=torch.bool, device=DEV)
            inside[top[top < keep]] = False
            to = torch.arange(keep, device=DEV)[inside]
            kv[blk[to], 0, h, tok[to]] = kv[blk[late], 0, h, tok[late]]
            v = kv[:, 1, h].view(-1, hd, page)
            v[blk[to], :, tok[to]] = v[blk[late], :, tok[late]]
            w[blk[to], h, tok[to]], pos[blk[to], h, tok[to]] = w[blk[late], h, tok[late]], pos[blk[late], h, tok[late]]
    return {"lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device=DEV), "kv": kv.double(), "key_pos": pos, "weights": w.double()}
