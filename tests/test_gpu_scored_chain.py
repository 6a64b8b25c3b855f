"""The cache with a budget as a server uses it: prompts in chunks with tracked weights, eviction, decode steps, tables of any width; attention against 64 bits over what the cache holds."""
import pytest
import torch

from rtp_llm_amd import kvcache, ops
from rtp_llm_amd.attention import AttentionConfigs, AttnImplFactory, LayerKVCache, PyAttentionInputs
from tests.scored_util import attend, bounds, evict, gather_plane

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rotation(most, hd):
    ang = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * 0.7 ** torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def held(cache, bt, b, n):
    """K, V (64 bits, [nkv, n, hd]) of a sequence's first n slots as the cache holds them."""
    kv, sc = cache.kv_cache_base, cache.kv_scale_base
    nblk, _, nkv, page, hd = kv.shape
    at = bt[b].long()
    k = kv[at, 0].permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :n]
    v = kv.reshape(nblk, 2, nkv, hd, page)[at, 1].permute(1, 0, 3, 2).reshape(nkv, -1, hd)[:, :n]
    if sc is None:
        return k.double(), v.double()
    s = sc.reshape(nblk, 2, nkv, page)[at].permute(1, 2, 0, 3).reshape(2, nkv, -1)[:, :, :n].double()
    code = lambda x: ((x.to(torch.int16) & 255) - 128).double()
    return code(k) * s[0, ..., None], code(v) * s[1, ..., None]


def empty_cache(blocks, nkv, page, hd, int8, dtype):
    kv, sc = kvcache.alloc_layer_cache(blocks, nkv, page, hd, int8, DEV, dtype)
    kv.zero_()
    if sc is not None:
        sc.fill_(1.0)
    return LayerKVCache(kv, sc, page, 0, *kvcache.alloc_planes(blocks, nkv, page, DEV))


def check_rows(q, out, cache, bt, b, lo, hi, n, cfg, old, *, scale, positions=None):
    """Rows of one sequence against 64 bits over the n slots that the cache holds: outputs, and the weights of all n slots (old: what they were)."""
    key_pos = gather_plane(cache.key_pos, bt, b, n) if cfg.slopes is not None else None
    ref, _, w, pv, size = attend(q, *held(cache, bt, b, n), lo, hi, scale=scale, cap=cfg.softcap, slopes=cfg.slopes, positions=positions, key_pos=key_pos)
    t_out, _, rel = bounds(q.dtype, q.shape[2], n, pv, size, ref)
    assert bool(((out.double() - ref).abs() <= t_out).all()), (b, float(((out.double() - ref).abs() / t_out).max()))
    want, have = old.double() * cfg.kv_decay + w, gather_plane(cache.weights, bt, b, n).double()
    t_w = w * (float(rel.max()) + q.shape[0] * q.shape[1] // w.shape[0] * 2.0 ** -24) + 2.0 ** -22 * want + q.shape[0] * 2.0 ** -60
    assert bool(((have - want).abs() <= t_w).all()), (b, float(((have - want).abs() / t_w).max()))


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("budget,blocks,max_seq_len,start", [(40, 4, 4096, 3000), (96, 8, 64, 50), (40, 300, 100, 0)])
def test_tables_of_any_width(dtype, int8, budget, blocks, max_seq_len, start):
    """A table as wide as the budget needs while positions are in the thousands, and tables whose slots go past the configuration's max_seq_len: every token that was written is attended and ranked."""
    nh, nkv, hd, page, B = 8, 2, 64, 16, 2
    c = AttentionConfigs(nh, nkv, hd, rope_dim=hd, max_seq_len=max_seq_len, kv_budget=budget, kv_sinks=2, kv_recent=8, kv_decay=0.9)
    cs = rotation(4096, hd)
    cache = empty_cache(B * blocks + 1, nkv, page, hd, int8, dtype)
    bt = (torch.randperm(B * blocks, generator=torch.Generator().manual_seed(3)) + 1).reshape(B, blocks).int().to(DEV)
    lens, positions = torch.zeros(B, dtype=torch.int32), torch.full((B,), start, dtype=torch.int32)
    g = torch.Generator(device=DEV).manual_seed(budget)
    for step in range(130):
        impl = AttnImplFactory.get_fmha_impl(c, PyAttentionInputs(sequence_lengths=lens, kv_cache_kernel_block_id_device=bt, token_positions=positions), cos_sin=cs)
        qkv = torch.randn(B, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
        n = int(lens[0]) + 1
        old = [gather_plane(cache.weights, bt, b, n).clone() for b in range(B)]
        out = impl.forward(qkv, cache).view(B, nh, hd)
        scratch = empty_cache(B * blocks + 1, nkv, page, hd, int8, dtype) if step == 0 else scratch
        q = ops.rope_kv_write_slots(qkv, None, cs, impl.positions, impl.slots, bt, scratch.kv_cache_base, scratch.kv_scale_base, nh, nkv, hd, page)     # the rotated queries
        for b in range(B):
            old[b][:, n - 1] = 0
            check_rows(q[b:b + 1], out[b:b + 1], cache, bt, b, torch.zeros(1, device=DEV), torch.full((1,), n, device=DEV), n, c, old[b], scale=hd ** -0.5)
            assert gather_plane(cache.key_pos, bt, b, n)[:, -1].tolist() == [start + step] * nkv
        lens, positions = lens + 1, positions + 1
        if n == min(blocks * page, budget + 24):
            assert impl.evict(cache).tolist() == [budget] * B
            lens = torch.full((B,), budget, dtype=torch.int32)
            for b in range(B):                                               # the first and the newest are all there
                kept = gather_plane(cache.key_pos, bt, b, budget)
                assert all({start, start + 1, *range(start + step - 7, start + step + 1)} <= set(row) or start > 1 and {*range(start + step - 7, start + step + 1)} <= set(row) for row in kept.tolist())


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("nh,nkv,hd,page,form", [(28, 4, 128, 16, "cap"), (14, 2, 64, 32, "slopes")])
def test_prompts_then_evictions_then_steps(nh, nkv, hd, page, form, dtype, int8):
    """Prompts of unequal length in two portions (written, attended, weights kept), a first eviction, then steps of one token with evictions between."""
    B, budget, portions = 3, 64, ([70, 33, 100], [41, 90, 2])
    G = nh // nkv
    slopes = torch.tensor([0.5 ** (1 + 7 * h / nh) for h in range(nh)], device=DEV) if form == "slopes" else None
    c = AttentionConfigs(nh, nkv, hd, rope_dim=hd, max_seq_len=256, kv_budget=budget, kv_sinks=4, kv_recent=16, kv_decay=0.95, softcap=20.0 if form == "cap" else 0.0, slopes=slopes)
    cs = None if form == "slopes" else rotation(256, hd)
    M = -(-160 // page)
    cache = empty_cache(B * M + 1, nkv, page, hd, int8, dtype)
    kv, sc = cache.kv_cache_base, cache.kv_scale_base
    bt = torch.randperm(B * M + 1, generator=torch.Generator().manual_seed(4))[: B * M].reshape(B, M).int().to(DEV)
    g = torch.Generator(device=DEV).manual_seed(nh)
    have = [0] * B
    for rows in portions:
        start = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
        slots = torch.cat([torch.arange(h, h + r, device=DEV) for h, r in zip(have, rows)]).int()
        seq = torch.cat([torch.full((r,), b, device=DEV) for b, r in enumerate(rows)]).int()
        qkv = torch.randn(sum(rows), (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
        old = [gather_plane(cache.weights, bt, b, have[b] + rows[b]).clone() for b in range(B)]
        q = ops.rope_kv_write_slots(qkv, None, cs, slots, slots, bt, kv, sc, nh, nkv, hd, page, row_seq=seq, key_pos=cache.key_pos, weights=cache.weights)
        out = ops.paged_attention_scored(q, kv, sc, bt, slots + 1, nkv, page, M * page, row_start=start, q_len=max(rows), softcap=c.softcap, slopes=slopes,
                                         positions=slots if slopes is not None else None, key_pos=cache.key_pos if slopes is not None else None, weights=cache.weights, decay=c.kv_decay).view(-1, nh, hd)
        for b in range(B):
            at, n = slice(int(start[b]), int(start[b + 1])), have[b] + rows[b]
            old[b][:, have[b]:] = 0
            check_rows(q[at], out[at], cache, bt, b, torch.zeros(rows[b], device=DEV), slots[at] + 1, n, c, old[b], scale=hd ** -0.5, positions=slots[at])
            have[b] = n
    lens, positions = torch.tensor(have, dtype=torch.int32), torch.tensor(have, dtype=torch.int32)
    lens_dev = lens.to(DEV)

    def moves(new_of, n_of, newest):
        """An eviction against the definition's moves: positions, and keys and values of every kept slot."""
        before = [(gather_plane(cache.weights, bt, b, n_of[b]).tolist(), gather_plane(cache.key_pos, bt, b, n_of[b]).tolist(), *held(cache, bt, b, n_of[b])) for b in range(B)]
        new = new_of().tolist()
        assert new == [min(n, budget) for n in n_of]
        for b, (w, pos, k, v) in enumerate(before):
            for h in range(nkv):
                slot = list(range(n_of[b]))
                for s, d in evict(w[h], pos[h], n_of[b], budget, newest[b], c.kv_sinks, c.kv_recent):
                    slot[d] = s
                slot = slot[: new[b]]
                now_k, now_v = held(cache, bt, b, new[b])
                assert torch.equal(now_k[h], k[h, slot]) and torch.equal(now_v[h], v[h, slot])
                assert gather_plane(cache.key_pos, bt, b, new[b])[h].tolist() == [pos[h][s] for s in slot]
        return new

    nxt = positions.to(DEV)
    new = moves(lambda: ops.kv_evict(cache.weights, cache.key_pos, bt, lens_dev, nxt, kv, sc, budget, sinks=c.kv_sinks, recent=c.kv_recent), have, positions.tolist())
    lens = torch.tensor(new, dtype=torch.int32)
    for step in range(24):
        impl = AttnImplFactory.get_fmha_impl(c, PyAttentionInputs(sequence_lengths=lens, kv_cache_kernel_block_id_device=bt, token_positions=positions), cos_sin=cs)
        qkv = torch.randn(B, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
        n_of = [int(n) + 1 for n in lens]
        old = [gather_plane(cache.weights, bt, b, n_of[b]).clone() for b in range(B)]
        out = impl.forward(qkv, cache).view(B, nh, hd)
        spare = [x if x is None else x.clone() for x in (kv, sc)]
        q = ops.rope_kv_write_slots(qkv, None, cs, impl.positions, impl.slots, bt, *spare, nh, nkv, hd, page)
        for b in range(B):
            old[b][:, -1] = 0
            check_rows(q[b:b + 1], out[b:b + 1], cache, bt, b, torch.zeros(1, device=DEV), torch.full((1,), n_of[b], device=DEV), n_of[b], c, old[b], scale=hd ** -0.5,
                       positions=impl.positions[b:b + 1])
        lens, positions = lens + 1, positions + 1
        if step % 8 == 7:
            lens = torch.tensor(moves(lambda: impl.evict(cache), [int(n) for n in lens], positions.tolist()), dtype=torch.int32)
    assert G * nkv == nh
