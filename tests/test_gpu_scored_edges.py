"""Edges of scored attention, tracked writes and eviction: scores that are all -inf, rows whose intervals lie far apart under distance biases, the largest position, blocks outside the pool."""
import pytest
import torch

from rtp_llm_amd import ops
from tests import test_gpu_scored_attn as scored_attn
from tests.scored_util import attend, bounds, gather_plane, make_cache
from tests.test_gpu_scored_attn import run_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)]


def weight_bound(w, old, rel, terms, rows):
    """As the attention's other tests: each probability is off by rel, the sum of `terms` rounds at each, decay and addition once each, and what lies below 2^-60 of one may be lost."""
    return w * (rel + terms * 2.0 ** -24) + 2.0 ** -22 * (old + w) + rows * 2.0 ** -60


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("rows", [2, 5, 40, 700])
def test_scores_that_are_all_minus_infinity(nh, nkv, hd, dtype, int8, rows):
    """Row 0 sees slots 20 to 23 alone, whose scores are -inf: a softmax of these is not a number, in its output and in the weights of the slots it sees, and nowhere else.  The other rows see all
    slots: their shares of 20 to 23 are 0."""
    n, page = 60, 16
    g = torch.Generator(device=DEV).manual_seed(rows)
    kv, sc, bt, dense = make_cache([n], nkv, hd, page, dtype, int8, g, DEV)
    q = (torch.randn(rows, nh, hd, device=DEV, generator=g).abs() + 0.1).to(dtype)        # positive, the four keys negative: no inf - inf inside a score
    for t in range(20, 24):
        blk, o = int(bt[0, t // page]), t % page
        if int8:
            kv[blk, 0, :, o], sc[blk, 0, :, o] = 127, float("inf")                         # the stored byte of the code -1
        else:
            kv[blk, 0, :, o], kv[blk, 0, :, o, 3] = -1.0, float("-inf")
    begin, end = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.full((rows,), n, dtype=torch.int32, device=DEV)
    begin[0], end[0] = 20, 24
    w = torch.full((kv.shape[0], nkv, page), 0.5, device=DEV)
    out, lse = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, bt.shape[1] * page, begin=begin, q_len=rows, weights=w, return_lse=True)
    out, got = out.view(rows, nh, hd).double(), gather_plane(w, bt, 0, n).double()
    others = torch.tensor([t for t in range(n) if not 20 <= t < 24], device=DEV)
    k, v = (x[:, others].contiguous() for x in dense[0])
    ref, ref_lse, want, pv, size = attend(q[1:], k, v, torch.zeros(rows - 1, device=DEV), torch.full((rows - 1,), n, device=DEV), scale=hd ** -0.5)
    t_out, t_lse, rel = bounds(dtype, hd, n, pv, size, ref)
    assert bool(torch.isnan(out[0]).all()) and not bool(torch.isfinite(lse[0]).any())
    assert bool(((out[1:] - ref).abs() <= t_out).all()) and bool(((lse[1:].double() - ref_lse).abs() <= t_lse + 2.0 ** -22 * ref_lse.abs()).all())
    assert bool(torch.isnan(got[:, 20:24]).all())
    t_w = weight_bound(want, 0.5, float(rel.max()), rows * nh // nkv, rows)
    assert bool(((got[:, others] - 0.5 - want).abs() <= t_w).all())


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("nh,nkv,rows,gap", [(2, 1, 2, 60000), (4, 1, 8, 60000), (4, 1, 40, 60000), (1, 1, 24, 50000)])
def test_biases_of_rows_that_see_slots_far_apart(nh, nkv, rows, gap, dtype, int8, planes):
    """One half of a sequence's rows sees 40 slots at its start, the other half 40 a long way behind, both next to the rows' positions: biases are small in every row, and scores as exact as those of either
    half alone."""
    hd, page = 64, 64
    n = gap + 40
    g = torch.Generator(device=DEV).manual_seed(rows)
    kv, sc, bt, dense = make_cache([n], nkv, hd, page, dtype, int8, g, DEV)
    q = torch.randn(rows, nh, hd, device=DEV, generator=g).to(dtype)
    late = torch.arange(rows, device=DEV) % 2 == 1
    begin, end = torch.where(late, gap, 0).int(), torch.where(late, n, 40).int()
    positions, slopes = end + 2, torch.tensor([0.5 ** (1 + h) for h in range(nh)], device=DEV)
    key_pos = None
    if planes:                                                                # the slots' numbers, kept beside the cache
        key_pos = torch.zeros(kv.shape[0], nkv, page, dtype=torch.int32, device=DEV)
        key_pos[bt[0].long()] = torch.arange(bt.shape[1] * page, device=DEV).int().view(-1, 1, page).expand(-1, nkv, -1)
    w = torch.zeros(kv.shape[0], nkv, page, device=DEV)
    out, lse = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, bt.shape[1] * page, begin=begin, q_len=rows, slopes=slopes, positions=positions, key_pos=key_pos, weights=w, decay=0.0,
                                          return_lse=True)
    out, got = out.view(rows, nh, hd).double(), gather_plane(w, bt, 0, n).double()
    for half, first in ((~late, 0), (late, gap)):
        k, v = (x[:, first:first + 40].contiguous() for x in dense[0])
        m = int(half.sum())
        ref, ref_lse, want, pv, size = attend(q[half], k, v, torch.zeros(m, device=DEV), torch.full((m,), 40, device=DEV), scale=hd ** -0.5, slopes=slopes, positions=positions[half] - first)
        t_out, t_lse, rel = bounds(dtype, hd, 40, pv, size, ref)
        assert bool(((out[half] - ref).abs() <= t_out).all()), float(((out[half] - ref).abs() / t_out).max())
        diff = (lse[half].double() - ref_lse).abs()
        assert bool((diff <= t_lse + 2.0 ** -22 * ref_lse.abs()).all()), float(diff.max())
        t_w = weight_bound(want, 0.0, float(rel.max()), m * nh // nkv, rows)
        assert bool(((got[:, first:first + 40] - want).abs() <= t_w).all()), float(((got[:, first:first + 40] - want).abs() / t_w).max())
    assert bool((got[:, 40:gap] == 0).all())


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("T", [1, 70])
def test_unrotated_rows_take_every_position(T, dtype, int8):
    """Without a rotation any position from 0 to 2^31 - 1 is kept with its row; below 0 a row is out of range."""
    nh, nkv, hd, page = 4, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(T)
    M = -(-T // page)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
    bt, slots = torch.arange(M, dtype=torch.int32, device=DEV).view(1, M), torch.arange(T, dtype=torch.int32, device=DEV)
    for p, lost in (((1 << 31) - 1, 0), ((1 << 31) - 2, 0), (0, 0), (-1, T), (-(1 << 31), T)):
        kv = torch.zeros(M, 2, nkv, page, hd, device=DEV, dtype=torch.int8 if int8 else dtype)
        sc = torch.zeros(M, 2, nkv, page, device=DEV) if int8 else None
        pos, w, oob = torch.full((M, nkv, page), 7, dtype=torch.int32, device=DEV), torch.ones(M, nkv, page, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.rope_kv_write_slots(qkv, None, None, torch.full((T,), p, dtype=torch.int32, device=DEV), slots, bt, kv, sc, nh, nkv, hd, page, q_len=T, key_pos=pos, weights=w, oob_count=oob)
        assert int(oob) == lost, p
        kept, cap = gather_plane(pos, bt, 0, M * page), M * page
        assert bool((kept[:, :T] == (7 if lost else p)).all()) and bool((kept[:, T:] == 7).all()), p
        assert bool((gather_plane(w, bt, 0, cap)[:, :T] == (1 if lost else 0)).all())
        assert bool((kv != 0).any()) == (not lost)


@pytest.mark.parametrize("rows,nh", [(1, 4), (6, 4), (40, 4), (700, 4)])
@pytest.mark.parametrize("int8", [False, True])
def test_weights_of_blocks_outside_the_pool_are_not_written(rows, nh, int8):
    """Ids that are no blocks read the pool's first or last block in place; no plane entry of those two, or of any block that the table does not name, changes.  700 rows: 1400 columns a head, whose
    shares are added by a launch of their own."""
    nkv, hd, page, nblk = 2, 64, 16, 12
    g = torch.Generator(device=DEV).manual_seed(rows)
    if int8:
        kv, sc = torch.randint(-128, 128, (nblk, 2, nkv, page, hd), generator=g, device=DEV, dtype=torch.int8), torch.rand(nblk, 2, nkv, page, device=DEV, generator=g) * 0.02
    else:
        kv, sc = torch.randn(nblk, 2, nkv, page, hd, device=DEV, generator=g).half(), None
    bt = torch.tensor([[3, -7, 5, 1 << 30, 6], [-(1 << 31), 7, 12, 8, 9]], dtype=torch.int32, device=DEV)
    w = torch.rand(nblk, nkv, page, device=DEV, generator=g)
    before = w.clone()
    q = torch.randn(2 * rows, nh, hd, device=DEV, generator=g).half()
    end = torch.tensor([73] * rows + [80] * rows, dtype=torch.int32, device=DEV)
    out = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, 80, q_len=rows, weights=w)
    assert bool(torch.isfinite(out.float()).all()) and bool(torch.isfinite(w).all())
    named = [3, 5, 6, 7, 8, 9]
    rest = [i for i in range(nblk) if i not in named]
    assert torch.equal(w[rest], before[rest])
    changed = w != before
    assert bool(changed[[3, 5, 7, 8, 9]].all()) and bool(changed[6, :, :9].all()) and not bool(changed[6, :, 9:].any())


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("cap,bias,mask", [(0.0, None, "causal"), (30.0, None, "window"), (0.0, "slots", "prefix"), (20.0, "planes", "causal"), (0.0, None, "documents")])
def test_chunks_behind_long_contexts(nh, nkv, hd, dtype, int8, cap, bias, mask):
    """A portion of a long prompt: more than 8192 slots, more than 128 columns a head, odd sizes."""
    run_case(nh, nkv, hd, 16, dtype, int8, [8301, 250], [67, 33], mask, cap, bias, True, decay=0.5)


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,rows", [(28, 4, 128, 3), (28, 4, 128, 4), (14, 2, 64, 4), (16, 2, 128, 4)])
@pytest.mark.parametrize("cap,bias,mask", [(0.0, "planes", "window"), (15.0, None, "causal")])
def test_few_rows_in_two_tiles(monkeypatch, nh, nkv, hd, rows, dtype, int8, cap, bias, mask):
    """17 to 32 columns a head, sequences of unequal length.
    Random positions set scores hundreds apart: a row of two slots can draw 2^-133 of one beside a value of exactly 0.  What a product of a probability (and, 8 bits, a value's scale) has below 2^-126, the
    smallest normal number of fp32 and bf16, may be 0: with codes up to 2^7, 16-bit values up to 2^3, at most 2^-119 a slot."""
    def with_smallest(dtype, hd, L, pv, size, out):
        t_out, t_lse, rel = bounds(dtype, hd, L, pv, size, out)
        return t_out + L * 2.0 ** -119, t_lse, rel
    monkeypatch.setattr(scored_attn, "bounds", with_smallest)
    run_case(nh, nkv, hd, 32, dtype, int8, [500, 0, 77, 1200], [rows, rows - 1, 1, rows], mask, cap, bias, True)
