"""Paged attention with score forms against 64-bit attention over the same pages: caps, distance biases, intervals of every kind, rows that see nothing, lengths of 0 and 1, odd pages,
garbage behind the context, 8- and 16-bit caches, any group of heads, accumulated weights."""
import pytest
import torch

from rtp_llm_amd import _C, ops
from tests.scored_util import attend, bounds, gather_plane, make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS = [(28, 4, 128, 16), (14, 2, 64, 64), (8, 8, 128, 48), (8, 2, 64, 16), (6, 2, 64, 32), (71, 1, 64, 16), (40, 2, 128, 80), (16, 1, 128, 16)]


def run_case(nh, nkv, hd, page, dtype, int8, ctx, rows, mask, cap, bias, track, *, decay=1.0, lse=True, seed=0, qscale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + nh + hd)
    B, n = len(ctx), max(rows)
    L = [c + r for c, r in zip(ctx, rows)]
    kv, sc, bt, dense = make_cache(L, nkv, hd, page, dtype, int8, g, DEV)
    T = sum(rows)
    start = torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    wide = (torch.randn(T, nh * hd + 64, device=DEV, generator=g) * qscale).to(dtype)
    q = wide[:, : nh * hd].unflatten(1, (nh, hd))
    slot = torch.cat([torch.arange(c, c + r, device=DEV) for c, r in zip(ctx, rows)]).int()
    size = torch.cat([torch.full((r,), l, device=DEV) for l, r in zip(L, rows)]).int()
    end, begin = slot + 1, None
    if mask == "window":
        begin = (end - 37).int()                                            # negative ones are from 0 on
    elif mask == "documents":
        begin = (slot // 50 * 50).int()
    elif mask == "prefix":
        end = torch.maximum(end, size // 2).int()
    elif mask == "holes":                                                   # rows that see nothing, rows that see one slot, ends far beyond the cache
        end, begin = end.clone(), torch.zeros_like(end)
        begin[::3] = end[::3]
        begin[1::5] = end[1::5] - 1
        end[2::7] = -5
    slopes = positions = key_pos = None
    if bias:
        slopes = torch.tensor([0.5 ** (1 + 7 * h / nh) for h in range(nh)], device=DEV)
        positions = slot + (3 if bias == "planes" else 0)
        if bias == "planes":
            key_pos = torch.randint(0, max(L) + 1, kv.shape[:1] + (nkv, page), generator=g, device=DEV, dtype=torch.int32)
    weights = torch.rand(kv.shape[0], nkv, page, device=DEV, generator=g) if track else None
    before = None if weights is None else weights.clone()
    M = bt.shape[1]
    out, got_lse = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, M * page, begin=begin, row_start=start, q_len=n, softcap=cap, slopes=slopes, positions=positions,
                                              key_pos=key_pos, weights=weights, decay=decay, return_lse=True)
    out = out.view(T, nh, hd).double()
    untouched = torch.ones_like(before, dtype=torch.bool) if track else None
    for b in range(B):
        r0, r1 = int(start[b]), int(start[b + 1])
        if r1 == r0:
            continue
        lo = torch.zeros(r1 - r0, device=DEV) if begin is None else begin[r0:r1].clamp_min(0)
        ref, ref_lse, w, pv, sz = attend(q[r0:r1], *dense[b], lo, end[r0:r1], scale=hd ** -0.5, cap=cap, slopes=slopes, positions=None if positions is None else positions[r0:r1],
                                         key_pos=None if key_pos is None else gather_plane(key_pos, bt, b, L[b]))
        t_out, t_lse, rel = bounds(dtype, hd, L[b], pv, sz, ref)
        assert bool(((out[r0:r1] - ref).abs() <= t_out).all()), ("out", b, float(((out[r0:r1] - ref).abs() / t_out).max()))
        empty = ~torch.isfinite(ref_lse)
        assert bool((out[r0:r1][empty] == 0).all()) and bool((got_lse[r0:r1][empty] == float("-inf")).all())
        diff = (got_lse[r0:r1].double() - ref_lse).masked_fill(empty, 0).abs()
        assert bool((diff <= t_lse + 2.0 ** -22 * ref_lse.masked_fill(empty, 0).abs()).all()), ("lse", b, float(diff.max()))
        if track:
            hi = end[r0:r1].clamp(0, L[b])
            reach = int(hi.masked_fill(hi <= lo, 0).max())                  # of the rows that see something
            old = gather_plane(before, bt, b, reach).double() * decay
            want, have = old + w[:, :reach], gather_plane(weights, bt, b, reach).double()
            t_w = w[:, :reach] * (float(rel.max()) + (r1 - r0) * nh // nkv * 2.0 ** -24) + 2.0 ** -22 * want + (r1 - r0) * 2.0 ** -60
            assert bool(((have - want).abs() <= t_w).all()), ("weights", b, float(((have - want).abs() / t_w.clamp_min(1e-30)).max()))
            for t in range(reach):
                untouched[int(bt[b, t // page]), :, t % page] = False
    if track:
        assert torch.equal(weights[untouched], before[untouched])           # slots behind the rows' ends and other pages
    return out


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("nh,nkv,hd,page", HEADS)
@pytest.mark.parametrize("cap,bias,mask,track", [(0.0, None, "causal", False), (5.0, None, "window", True), (0.0, "slots", "causal", True), (30.0, "planes", "holes", True)])
def test_decode(nh, nkv, hd, page, dtype, int8, cap, bias, mask, track):
    run_case(nh, nkv, hd, page, dtype, int8, [0, 1, 15, 16, 100, 333], [1] * 6, mask, cap, bias, track)


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("nh,nkv,hd,page", HEADS)
@pytest.mark.parametrize("cap,bias,mask,track", [(0.0, None, "causal", True), (5.0, None, "window", False), (0.0, "slots", "documents", True), (30.0, "planes", "prefix", True), (0.0, None, "holes", True)])
def test_chunks(nh, nkv, hd, page, dtype, int8, cap, bias, mask, track):
    run_case(nh, nkv, hd, page, dtype, int8, [0, 70, 5, 0], [130, 33, 0, 1], mask, cap, bias, track, decay=0.5)


@pytest.mark.parametrize("rows", [2, 3, 4, 5, 8, 9, 17, 40])
@pytest.mark.parametrize("int8", [False, True])
def test_few_rows(rows, int8):
    run_case(28, 4, 128, 16, torch.float16, int8, [257, 30], [rows, max(1, rows - 1)], "causal", 20.0, "slots", True)


@pytest.mark.parametrize("nh,nkv,hd,ctx,B,rows", [(8, 1, 128, 20000, 1, 1), (28, 4, 128, 5000, 2, 1), (8, 1, 128, 9000, 1, 40), (14, 2, 64, 3000, 70, 1), (8, 1, 128, 3000, 40, 3)])
@pytest.mark.parametrize("int8", [False, True])
def test_long(nh, nkv, hd, ctx, B, rows, int8):
    """Few rows over long contexts (the keys are split over blocks) and many sequences (they are not)."""
    run_case(nh, nkv, hd, 16, torch.float16, int8, [max(0, ctx - 97 * b) for b in range(B)], [rows] * B, "causal", 30.0, None, True)


@pytest.mark.parametrize("nh,nkv,int8", [(4, 1, False), (8, 4, False), (8, 4, True)])
@pytest.mark.parametrize("rows", [1, 2])
def test_many_short_sequences(nh, nkv, int8, rows):
    """300 sequences, some without tokens or rows: in runs that cross sequences (one kv head), and a block for each pair (four)."""
    ctx = [(37 * b) % 211 if b % 5 else 0 for b in range(300)]
    run_case(nh, nkv, 64, 16, torch.float16, int8, ctx, [0 if b % 7 == 3 else 1 + b % rows for b in range(300)], "window", 0.0, None, True)


def test_large_scores_and_late_maxima():
    """Scores that grow along the keys (the running maximum moves all the time) and reach hundreds, capped and not."""
    for cap in (0.0, 50.0):
        run_case(8, 2, 128, 16, torch.bfloat16, False, [700, 64], [3, 33], "causal", cap, "slots", True, qscale=40.0)


def test_decay_zero_overwrites_what_is_not_a_number():
    g = torch.Generator(device=DEV).manual_seed(4)
    kv, sc, bt, dense = make_cache([50], 2, 64, 16, torch.float16, False, g, DEV)
    q = torch.randn(1, 4, 64, device=DEV, generator=g).half()
    w = torch.full((kv.shape[0], 2, 16), float("nan"), device=DEV)
    end = torch.tensor([50], dtype=torch.int32, device=DEV)
    ops.paged_attention_scored(q, kv, sc, bt, end, 2, 16, 64, weights=w, decay=0.0)
    _, _, want, _, _ = attend(q, *dense[0], torch.zeros(1, device=DEV), end, scale=64 ** -0.5)
    assert torch.allclose(gather_plane(w, bt, 0, 50).double(), want, rtol=1e-5, atol=1e-9)
    assert int(torch.isnan(w).sum()) == w.numel() - 100


def test_block_ids_out_of_the_pool_are_clamped():
    """Ids that are not blocks give wrong rows, never another address; their weights are not written."""
    g = torch.Generator(device=DEV).manual_seed(5)
    kv, sc, bt, _ = make_cache([40, 64], 2, 64, 16, torch.float16, False, g, DEV, fill=0.0)
    bad = bt.clone()
    bad[0, 1], bad[1, 0] = -7, 1 << 30
    w = torch.zeros(kv.shape[0], 2, 16, device=DEV)
    q = torch.randn(2, 4, 64, device=DEV, generator=g).half()
    ops.paged_attention_scored(q, kv, sc, bad, torch.tensor([40, 64], dtype=torch.int32, device=DEV), 2, 16, 64, weights=w)
    q2 = torch.randn(2 * 40, 4, 64, device=DEV, generator=g).half()
    out = ops.paged_attention_scored(q2, kv, sc, bad, torch.full((80,), 40, dtype=torch.int32, device=DEV), 2, 16, 64, q_len=40, weights=w)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(w).all())


def test_row_starts_out_of_range_and_rows_behind_the_last():
    g = torch.Generator(device=DEV).manual_seed(6)
    kv, sc, bt, _ = make_cache([40, 64], 2, 64, 16, torch.float16, False, g, DEV, fill=0.0)
    for rows in (6, 60):
        q = torch.randn(rows, 4, 64, device=DEV, generator=g).half()
        end = torch.full((rows,), 30, dtype=torch.int32, device=DEV)
        out = torch.full((rows, 256), 9.0, dtype=torch.float16, device=DEV)
        ops.paged_attention_scored(q, kv, sc, bt, end, 2, 16, 64, row_start=torch.tensor([0, 1, rows - 2], dtype=torch.int32, device=DEV), q_len=rows, out=out)
        assert bool((out[rows - 2:] == 9.0).all()) and not bool((out[: rows - 2] == 9.0).all(1).any())
        for start in ([-3, 2, 1 << 30], [5, 1, 3], [1 << 30, 0, 1]):
            ops.paged_attention_scored(q, kv, sc, bt, end, 2, 16, 64, row_start=torch.tensor(start, dtype=torch.int32, device=DEV), q_len=rows, out=out)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 128, 16), (14, 2, 64, 48)])
@pytest.mark.parametrize("rows,n", [(3, 90), (70, 150), (300, 300)])
@pytest.mark.parametrize("what", ["value", "key"])
def test_what_is_not_finite_reaches_the_rows_that_see_it_alone(nh, nkv, hd, page, dtype, int8, rows, n, what):
    """Slots that hold infinities or NaN next to slots that others see: a row that sees none of them gets what it gets without them, one that sees them gets the formula's infinities and NaN in
    their channels (8 bits: a scale that is not a number, NaN in all), and the weights of slots that only untouched rows see stay as they were.
    Values: bit for bit.  Keys: 64 lanes' columns move their running maxima together, when one of them has grown by enough, so a neighbour's infinite score moves the point from which a
    column's exponentials are taken.  exp2(s - m) / sum exp2(s - m) does not depend on m, its roundings do: each run is within the formula's bounds, not the same as the other."""
    g = torch.Generator(device=DEV).manual_seed(rows + hd)
    kv, sc, bt, dense = make_cache([n], nkv, hd, page, dtype, int8, g, DEV)
    q = torch.randn(rows, nh, hd, device=DEV, generator=g).to(dtype)
    r = torch.arange(rows, device=DEV)
    end = (n - rows + 1 + r).int()
    begin = torch.where(r % 3 == 0, torch.zeros_like(end), (end - 20).clamp_min(0)).int()
    begin[1::7] = end[1::7]                                                  # and rows that see nothing
    bad = {n // 2: float("inf"), n // 2 + 1: float("-inf"), n - 3: float("nan"), n - 30: float("inf")}

    def run():
        w = torch.full((kv.shape[0], nkv, page), 0.25, device=DEV)
        out, lse = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, bt.shape[1] * page, begin=begin, q_len=rows, weights=w, return_lse=True)
        return out.view(rows, nh, hd), lse, w

    clean, lse0, w0 = run()
    for t, x in bad.items():
        blk, o = int(bt[0, t // page]), t % page
        if int8:
            sc[blk, 0 if what == "key" else 1, :, o] = float("nan")
        elif what == "key":
            kv[blk, 0, :, o, 5] = x
        else:
            kv[blk, 1].view(nkv, hd, page)[:, 5, o] = x
    out, lse, w = run()
    sees = {t: (begin <= t) & (t < end) for t in bad}
    some = torch.stack(list(sees.values())).any(0)
    assert bool(some.any()) and (rows == 3 or bool((~some & (end > begin)).any()))
    gw, gw0 = gather_plane(w, bt, 0, n), gather_plane(w0, bt, 0, n)
    if what == "value":
        assert torch.equal(out[~some], clean[~some])
    ref, ref_lse, _, pv, size = attend(q, *dense[0], begin, end, scale=hd ** -0.5)
    t_out, t_lse, rel = bounds(dtype, hd, n, pv, size, ref)
    fine = ~some & (end > begin)
    assert bool(((out.double() - ref).abs() <= t_out)[~some].all())
    assert bool(((lse.double() - ref_lse).abs() <= t_lse + 2.0 ** -22 * ref_lse.abs())[fine].all()) and bool((lse[end <= begin] == float("-inf")).all())
    if what == "value":
        assert torch.equal(lse, lse0) and torch.equal(gw, gw0)               # scores do not look at values
        if int8:
            assert bool(torch.isnan(out[some]).all())
        else:
            rest = [d for d in range(hd) if d != 5]
            assert torch.equal(out[:, :, rest], clean[:, :, rest])
            up, down, nan = (torch.stack([sees[t] for t, x in bad.items() if k(x)]).any(0) for k in (lambda x: x == float("inf"), lambda x: x == float("-inf"), lambda x: x != x))
            got = out[:, :, 5]
            assert bool(torch.isnan(got[nan | (up & down)]).all()) and bool((~torch.isfinite(got[some])).all())
            assert not bool((got[up & ~down & ~nan] == float("-inf")).any()) and not bool((got[down & ~up & ~nan] == float("inf")).any())
    else:
        touched = torch.zeros(n, dtype=torch.bool, device=DEV)               # slots that some row sees which sees a bad one too
        for i in torch.nonzero(some).flatten().tolist():
            touched[int(begin[i]):int(end[i])] = True
        t_w = gw0.double() * (2 * float(rel[fine].max() if bool(fine.any()) else 0) + 2.0 ** -21 + rows * (nh // nkv) * 2.0 ** -23)      # two runs of the sums' bounds
        assert bool(((gw.double() - gw0.double()).abs() <= t_w)[:, ~touched].all())
        if int8:
            assert bool(torch.isnan(out[some]).all()) and bool(torch.isnan(gw[:, touched]).all())


@pytest.mark.parametrize("dtype,int8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("rows", [2, 4, 40])
def test_documents_side_by_side_keep_to_themselves(rows, dtype, int8):
    """Half the rows see [0, 40), half [60, 100): what the first document and the gap between them hold does not reach the second's rows, inside a tile of 32 or across."""
    nh, nkv, hd, page, n = 8, 4, 128, 16, 100
    g = torch.Generator(device=DEV).manual_seed(rows)
    kv, sc, bt, _ = make_cache([n], nkv, hd, page, dtype, int8, g, DEV)
    q = torch.randn(rows, nh, hd, device=DEV, generator=g).to(dtype)
    late = torch.arange(rows, device=DEV) >= rows // 2
    begin, end = torch.where(late, 60, 0).int(), torch.where(late, 100, 40).int()

    def run():
        w = torch.zeros(kv.shape[0], nkv, page, device=DEV)
        out, lse = ops.paged_attention_scored(q, kv, sc, bt, end, nkv, page, bt.shape[1] * page, begin=begin, q_len=rows, weights=w, return_lse=True)
        return out, lse, gather_plane(w, bt, 0, n)

    clean, lse0, w0 = run()
    for t in (10, 39, 40, 50, 59):
        blk, o = int(bt[0, t // page]), t % page
        if int8:
            sc[blk, :, :, o] = float("nan")
        else:
            kv[blk, 0, :, o], kv[blk, 1].view(nkv, hd, page)[:, :, o] = float("nan"), float("inf")
    out, lse, w = run()
    assert torch.equal(out[late], clean[late]) and torch.equal(lse[late], lse0[late]) and torch.equal(w[:, 40:], w0[:, 40:])
    assert bool(torch.isnan(out[~late]).all()) and bool(torch.isnan(lse[~late]).all()) and bool(torch.isnan(w[:, :40]).all())


@pytest.mark.parametrize("rows,track", [(1, True), (1, False), (48, True)])
def test_graphs_and_streams(rows, track):
    """Two captured calls of different sizes, replayed in turn with eager work between, and the same calls on two streams at once: every result is the eager one, bit for bit."""
    cases = []
    for i, (ctx, B) in enumerate(((900, 3), (4000, 1))):
        g = torch.Generator(device=DEV).manual_seed(20 + i)
        kv, sc, bt, _ = make_cache([ctx + rows] * B, 2, 128, 16, torch.float16, False, g, DEV)
        q = torch.randn(B * rows, 14, 128, device=DEV, generator=g).half()
        end = torch.cat([torch.arange(ctx + 1, ctx + rows + 1, device=DEV)] * B).int()
        w = torch.zeros(kv.shape[0], 2, 16, device=DEV) if track else None
        call = lambda q=q, kv=kv, bt=bt, end=end, w=w: ops.paged_attention_scored(q, kv, None, bt, end, 2, 16, bt.shape[1] * 16, q_len=rows, softcap=20.0, weights=w, decay=0.0, return_lse=True)
        cases.append((call, w))
    eager = []
    for call, w in cases:
        out, lse = call()
        eager.append((out.clone(), lse.clone(), None if w is None else w.clone()))
    torch.cuda.synchronize()
    graphs = []
    for call, _ in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = call()
        graphs.append((gr, res))
    same = lambda got, i, w: torch.equal(got[0], eager[i][0]) and torch.equal(got[1], eager[i][1]) and (w is None or torch.equal(w, eager[i][2]))
    for _ in range(4):
        for i, (gr, res) in enumerate(graphs):
            if cases[i][1] is not None:
                cases[i][1].fill_(7.0 if i else float("nan")).masked_fill_(eager[i][2] == 0, 0.0)
            gr.replay()
            assert same(cases[1 - i][0](), 1 - i, cases[1 - i][1])
            torch.cuda.synchronize()
            assert same(res, i, cases[i][1])
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for (call, _), s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], eager[i % 2][0]) and torch.equal(a[1], eager[i % 2][1]) for i, a in enumerate(got))


def test_the_same_as_plain_attention():
    """Without forms the call is the one the framework had: both within a rounding of the same result."""
    g = torch.Generator(device=DEV).manual_seed(9)
    kv, sc, bt, _ = make_cache([200, 77], 4, 128, 16, torch.float16, False, g, DEV)
    q = torch.randn(2, 28, 128, device=DEV, generator=g).half()
    lens = torch.tensor([200, 77], dtype=torch.int32, device=DEV)
    a = ops.paged_attention_scored(q, kv, sc, bt, lens, 4, 16, 208).float()
    b = ops.paged_decode_attention(q, kv, sc, bt, lens, 4, 16, 208).float()
    assert float((a - b).abs().max()) <= 2 * 2.0 ** -11 * 2 * 5
    assert int(_C.lib().mi355_abi_version()) == _C.ABI_VERSION
