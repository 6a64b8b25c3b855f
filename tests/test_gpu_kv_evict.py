"""Eviction by attention weight and the writer whose slot is not the position, against lists of moves from the definition: every cached byte, plane entry and length."""
import pytest
import torch

from rtp_llm_amd import ops
from tests.scored_util import evict, gather_plane, make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run_evict(L, keep, nkv, hd, page, dtype, int8, sinks, recent, *, values=None, shuffle=True, spoil=None, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kv, sc, bt, _ = make_cache(L, nkv, hd, page, dtype, int8, g, DEV, fill=0.0)
    if int8:
        sc = torch.rand(sc.shape, device=DEV, generator=g)
    nblk = kv.shape[0]
    w = torch.rand(nblk, nkv, page, device=DEV, generator=g) if values is None else values(nblk, nkv, page, g)
    pos = torch.zeros(nblk, nkv, page, dtype=torch.int32, device=DEV)
    nxt = []
    for b, n in enumerate(L):
        cap = bt.shape[1] * page
        p = torch.stack([torch.randperm(cap, generator=torch.Generator().manual_seed(h + 5)) if shuffle else torch.arange(cap) for h in range(nkv)]).int().to(DEV)
        pos[bt[b].long()] = p.view(nkv, -1, page).transpose(0, 1).contiguous()
        nxt.append(cap if shuffle else n)
    if spoil is not None:
        spoil(bt)
    before = [x if x is None else x.clone() for x in (kv, sc, w, pos)]
    lens = torch.tensor(L, dtype=torch.int32, device=DEV)
    new = ops.kv_evict(w, pos, bt, lens, torch.tensor(nxt, dtype=torch.int32, device=DEV), kv, sc, keep, sinks=sinks, recent=recent)
    assert new.tolist() == [min(n, keep) for n in L] and lens.tolist() == L
    want = [x if x is None else x.clone() for x in before]
    V = lambda x: x[:, 1].view(nblk, nkv, hd, page)
    for b, n in enumerate(L):
        bad = (lambda t, b=b: not 0 <= int(bt[b, t // page]) < nblk) if spoil is not None else None
        usable = bt[b].long().clamp(0, nblk - 1)
        for h in range(nkv):
            ww, pp = (x[usable, h].reshape(-1).tolist() for x in before[2:])
            for s, d in evict(ww, pp, n, keep, nxt[b], sinks, recent, bad):
                bs, bd, ts, td = int(bt[b, s // page]), int(bt[b, d // page]), s % page, d % page
                if not (0 <= bs < nblk and 0 <= bd < nblk):
                    continue
                want[0][bd, 0, h, td] = before[0][bs, 0, h, ts]
                V(want[0])[bd, h, :, td] = V(before[0])[bs, h, :, ts]
                if int8:
                    want[1][bd, :, h, td] = before[1][bs, :, h, ts]
                want[2][bd, h, td], want[3][bd, h, td] = before[2][bs, h, ts], before[3][bs, h, ts]
    for name, a, e in zip(("kv", "scale", "weights", "positions"), (kv, sc, w, pos), want):
        if a is not None:
            bits = lambda x: x.view(torch.int32) if x.dtype == torch.float32 else x.view(torch.int16) if x.element_size() == 2 else x
            assert torch.equal(bits(a), bits(e)), (name, int((bits(a) != bits(e)).sum()))


@pytest.mark.parametrize("nkv,hd,page,dtype,int8", [(4, 128, 16, torch.float16, False), (2, 64, 64, torch.bfloat16, False), (1, 128, 24, torch.float16, True), (8, 64, 32, torch.bfloat16, True), (3, 128, 40, torch.bfloat16, False)])
@pytest.mark.parametrize("keep,sinks,recent", [(64, 4, 16), (1, 0, 0), (100, 0, 100), (37, 37, 0), (250, 10, 3)])
def test_evict(nkv, hd, page, dtype, int8, keep, sinks, recent):
    run_evict([0, 1, 63, 64, 65, 300, 100, 251], keep, nkv, hd, page, dtype, int8, sinks, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "special"])
def test_ties_and_special_weights(kind):
    def values(nblk, nkv, page, g):
        if kind == "equal":
            return torch.full((nblk, nkv, page), 0.25, device=DEV)
        if kind == "few":
            return torch.randint(0, 3, (nblk, nkv, page), generator=g, device=DEV).float()
        if kind == "signs":
            return torch.randint(-2, 3, (nblk, nkv, page), generator=g, device=DEV).float() * torch.tensor([0.0, -0.0, 1.0, 2.0], device=DEV)[torch.randint(0, 4, (nblk, nkv, page), generator=g, device=DEV)]
        return torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, 1e-45, 3e38, -1.0], device=DEV)[torch.randint(0, 8, (nblk, nkv, page), generator=g, device=DEV)]
    run_evict([200, 333, 90], 77, 2, 64, 16, torch.float16, False, 3, 9, values=values)


def test_positions_in_order():
    run_evict([500, 129], 128, 4, 128, 16, torch.float16, False, 4, 32, shuffle=False)


@pytest.mark.parametrize("n", [5000, 40000])
def test_long(n):
    """Ranks kept in LDS, and formed again by every pass."""
    run_evict([n, n // 3], n // 2, 1, 64, 64, torch.float16, False, 4, 64, shuffle=False)


def test_blocks_out_of_the_pool_go_first_and_are_not_moved():
    def spoil(bt):
        bt[0, 2], bt[0, 5], bt[1, 0], bt[1, 3] = -1, 1 << 30, -(1 << 31), 99999
    run_evict([200, 120], 100, 2, 64, 16, torch.float16, False, 0, 0, spoil=spoil)


def test_a_budget_beyond_the_cache_changes_nothing():
    g = torch.Generator(device=DEV).manual_seed(5)
    kv, _, bt, _ = make_cache([70, 0, 33], 2, 64, 16, torch.float16, False, g, DEV, fill=0.0)
    w, pos = torch.rand(kv.shape[0], 2, 16, device=DEV, generator=g), torch.zeros(kv.shape[0], 2, 16, dtype=torch.int32, device=DEV)
    lens = torch.tensor([70, 0, 33], dtype=torch.int32, device=DEV)
    before = [x.clone() for x in (kv, w, pos)]
    for keep in (70, 96, 1 << 30):
        assert ops.kv_evict(w, pos, bt, lens, lens, kv, None, keep, sinks=4, recent=16).tolist() == [70, 0, 33]
        assert all(torch.equal(a, b) for a, b in zip((kv, w, pos), before))


@pytest.mark.parametrize("int8", [False, True])
def test_a_pool_of_more_than_32_bits_of_bytes(int8):
    """Write, attend (a row and many) and evict in blocks at the far end of a large pool: as in a small one."""
    nh, nkv, hd, page, n, far = 16, 8, 128, 16, 200, 270000 if int8 else 135000          # 8.8 GB
    g = torch.Generator(device=DEV).manual_seed(17)
    kv, sc, bt, _ = make_cache([n], nkv, hd, page, torch.float16, int8, g, DEV, fill=0.0)
    nblk, used = kv.shape[0], bt[0].long()
    w, pos = torch.rand(nblk, nkv, page, device=DEV, generator=g), torch.zeros(nblk, nkv, page, dtype=torch.int32, device=DEV)
    qkv = torch.randn(40, (nh + 2 * nkv) * hd, device=DEV, generator=g).half()
    big = torch.empty(far, *kv.shape[1:], dtype=kv.dtype, device=DEV)
    big_sc = torch.zeros(far, *sc.shape[1:], device=DEV) if int8 else None
    big_w, big_pos = torch.zeros(far, nkv, page, device=DEV), torch.zeros(far, nkv, page, dtype=torch.int32, device=DEV)
    for a, b in ((big, kv), (big_w, w), (big_pos, pos)) + (((big_sc, sc),) if int8 else ()):
        a[far - nblk:] = b
    assert big.numel() * big.element_size() > 1 << 33
    got = []
    for c, s, wt, ps, table in ((kv, sc, w, pos, bt), (big, big_sc, big_w, big_pos, bt + (far - nblk))):
        slots = torch.arange(n - 40, n, dtype=torch.int32, device=DEV)
        q = ops.rope_kv_write_slots(qkv, None, None, slots, slots, table, c, s, nh, nkv, hd, page, q_len=40, key_pos=ps, weights=wt)
        outs = [ops.paged_attention_scored(q, c, s, table, slots + 1, nkv, page, n, q_len=40, weights=wt), ops.paged_attention_scored(q[-1:], c, s, table, slots[-1:] + 1, nkv, page, n, weights=wt)]
        lens = torch.tensor([n], dtype=torch.int32, device=DEV)
        new = ops.kv_evict(wt, ps, table, lens, lens, c, s, 64, sinks=4, recent=16)
        at = table[0].long()
        got.append(outs + [new, c[at[:4]], wt[at[:4]], ps[at[:4]]] + ([s[at[:4]]] if int8 else []))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_graph_and_stream():
    """A captured eviction replayed over restored planes, with eager work between: the moves of the eager call."""
    g = torch.Generator(device=DEV).manual_seed(3)
    kv, _, bt, _ = make_cache([300, 220], 2, 128, 16, torch.float16, False, g, DEV, fill=0.0)
    w, pos = torch.rand(kv.shape[0], 2, 16, device=DEV, generator=g), torch.zeros(kv.shape[0], 2, 16, dtype=torch.int32, device=DEV)
    for b in range(2):
        pos[bt[b].long()] = torch.arange(bt.shape[1] * 16, device=DEV).int().view(-1, 1, 16).expand(-1, 2, -1)
    lens, nxt = torch.tensor([300, 220], dtype=torch.int32, device=DEV), torch.tensor([300, 220], dtype=torch.int32, device=DEV)
    start = [x.clone() for x in (kv, w, pos)]
    restore = lambda: [a.copy_(s) for a, s in zip((kv, w, pos), start)]
    call = lambda: ops.kv_evict(w, pos, bt, lens, nxt, kv, None, 128, sinks=4, recent=16)
    call()
    torch.cuda.synchronize()
    want = [x.clone() for x in (kv, w, pos)]
    assert not torch.equal(want[0], start[0])
    gr = torch.cuda.CUDAGraph()
    restore()
    with torch.cuda.graph(gr):
        new = call()
    for i in range(3):
        restore()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip((kv, w, pos), want)) and new.tolist() == [128, 128]
        restore()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, e) for a, e in zip((kv, w, pos), want))


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("nh,nkv,hd,page,T", [(28, 4, 128, 16, 5), (14, 2, 64, 64, 3), (28, 4, 128, 16, 300), (14, 2, 64, 24, 130), (71, 1, 64, 16, 70)])
@pytest.mark.parametrize("rotate", [True, False])
def test_write_slots(nh, nkv, hd, page, T, dtype, int8, rotate):
    """Against the writer that has one number for both: a row rotated at its position lands in its slot, planes beside it, padding and rows out of range nowhere."""
    g = torch.Generator(device=DEV).manual_seed(T)
    B, M = 3, -(-T // page) + 2
    nblk, cap, most = B * M + 1, M * page, 700
    bt = torch.randperm(nblk, generator=torch.Generator().manual_seed(2))[: B * M].reshape(B, M).int().to(DEV)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
    bias = torch.randn((nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
    ang = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * 0.9 ** torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float()
    seq = torch.randint(0, B, (T,), generator=g, device=DEV, dtype=torch.int32)
    slots = torch.randperm(cap, generator=g, device=DEV)[:T].int()
    positions = torch.randint(0, most, (T,), generator=g, device=DEV, dtype=torch.int32)
    lost = 0
    if T > 4:
        slots[0], slots[1], seq[2], seq[3] = -1, cap, B, -1
        lost = 3
        if rotate:
            positions[4] = most
        else:
            positions[4] = -2
        lost += 1
    new = lambda: (torch.zeros(nblk, 2, nkv, page, hd, device=DEV, dtype=torch.int8 if int8 else dtype), torch.ones(nblk, 2, nkv, page, device=DEV) if int8 else None)
    kv, sc = new()
    pos, w = torch.full((nblk, nkv, page), -9, dtype=torch.int32, device=DEV), torch.full((nblk, nkv, page), 5.0, device=DEV)
    oob = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = ops.rope_kv_write_slots(qkv, bias, cs if rotate else None, positions, slots, bt, kv, sc, nh, nkv, hd, page, row_seq=seq, key_pos=pos, weights=w, oob_count=oob)
    assert int(oob) == lost
    # the old writer, a row at a time in a pool whose table has the row's page at its position
    still = torch.tensor([[[1.0, 0.0]] * (hd // 2)] * most, device=DEV)
    want_kv, want_sc = new()
    want_pos, want_w = torch.full_like(pos, -9), torch.full_like(w, 5.0)
    for t in range(T):
        sl, sq, ps = int(slots[t]), int(seq[t]), int(positions[t])
        ok = 0 <= sl < cap and 0 <= sq < B and 0 <= ps < (most if rotate else 1 << 31)
        one_kv, one_sc = new()
        at = max(0, min(ps, most - 1))
        table = torch.zeros(1, most // page + 1, dtype=torch.int32, device=DEV)
        qq = ops.rope_kv_write(qkv[t:t + 1], bias, cs if rotate else still, torch.tensor([at], dtype=torch.int32, device=DEV), table, one_kv, one_sc, nh, nkv, hd, page)
        assert torch.equal(qq[0], q[t]), t
        if not ok:
            continue
        blk, i, j = int(bt[sq, sl // page]), sl % page, at % page
        want_kv[blk, 0, :, i] = one_kv[0, 0, :, j]
        want_kv[blk, 1].view(nkv, hd, page)[:, :, i] = one_kv[0, 1].view(nkv, hd, page)[:, :, j]
        if int8:
            want_sc[blk, :, :, i] = one_sc[0, :, :, j]
        want_pos[blk, :, i], want_w[blk, :, i] = ps, 0.0
    assert torch.equal(kv, want_kv) and torch.equal(pos, want_pos) and torch.equal(w, want_w)
    assert not int8 or torch.equal(sc, want_sc)
