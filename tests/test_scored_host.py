"""Refusals of the scored attention, the tracked writer and the eviction: on the host, before any launch."""
import ctypes as C
import random

import pytest
import torch

from rtp_llm_amd import _C, kvcache, ops
from tests.scored_util import evict


def _kv(**kw):
    d = dict(kv_base=16, scale_base=16, kv_dtype=_C.KV_FP16, page=16, nkv=4, hd=128, num_blocks=8, act_dtype=_C.ACT_F16)
    d.update(kw)
    return _C.KVLayer(*(d[k] for k, _ in _C.KVLayer._fields_))


def _attend(kv=None, *, q=16, ldq=28 * 128, table=16, M=4, starts=None, B=1, q_len=1, rows=1, nh=28, score=None, most=64, out=16, weights=None, decay=1.0, ws=16, nbytes=1 << 30):
    sc = score or _C.AttnScore(0.1, 0.0, None, None, None, None, 16)
    return _C.lib().mi355_paged_attn_scored(q, ldq, C.byref(kv or _kv()), table, M, starts, B, q_len, rows, nh, C.byref(sc), most, out, None, weights, decay, ws, nbytes, None)


@pytest.mark.parametrize("kw,said", [
    (dict(q=None), "null pointer"), (dict(out=None), "null pointer"), (dict(table=None), "null pointer"), (dict(score=_C.AttnScore(0.1, 0.0, None, None, None, None, None)), "null pointer"),
    (dict(kv=_kv(hd=96)), "hd=96"), (dict(kv=_kv(page=12)), "page=12"), (dict(kv=_kv(nkv=3)), "nkv=3"), (dict(kv=_kv(num_blocks=0)), "block table"), (dict(B=0), "B=0"),
    (dict(rows=2), "2 rows"), (dict(starts=16, rows=3), "3 rows"), (dict(ldq=28 * 128 - 8), "ldq"), (dict(ldq=28 * 128 + 4), "ldq"), (dict(most=65), "block table"), (dict(q=24), "16 bytes"),
    (dict(kv=_kv(kv_dtype=_C.KV_INT8, scale_base=None)), "scales"), (dict(kv=_kv(kv_dtype=_C.KV_BF16)), "kv_dtype"), (dict(kv=_kv(act_dtype=_C.ACT_F32)), "act_dtype"),
    (dict(score=_C.AttnScore(0.1, -1.0, None, None, None, None, 16)), "softcap"), (dict(score=_C.AttnScore(0.1, float("nan"), None, None, None, None, 16)), "softcap"),
    (dict(score=_C.AttnScore(0.1, 0.0, 16, None, None, None, 16)), "positions"), (dict(weights=16, decay=1.5), "decay"), (dict(weights=16, decay=float("nan")), "decay"),
    (dict(kv=_kv(num_blocks=1 << 26)), "2^31"), (dict(B=70000, rows=70000), "grid")])
def test_attention_refuses(kw, said):
    assert _attend(**kw) == _C.ERR_ARG
    assert said.encode() in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


@pytest.mark.parametrize("kw,said", [
    (dict(score=_C.AttnScore(0.0, 0.0, None, None, None, None, 16)), "scale=0"), (dict(score=_C.AttnScore(-0.1, 0.0, None, None, None, None, 16)), "scale=-0.1"),
    (dict(score=_C.AttnScore(float("nan"), 0.0, None, None, None, None, 16)), "scale"), (dict(score=_C.AttnScore(0.1, 1e-7, None, None, None, None, 16)), "softcap"),
    (dict(score=_C.AttnScore(0.1, 0.0, 16, 16, 24, None, 16)), "16 bytes"), (dict(ws=24), "16 bytes"), (dict(B=2048, rows=2048, nh=1 << 10, ldq=1 << 17, kv=_kv(nkv=1 << 10), M=1 << 20, most=1 << 24), "grid")])
def test_attention_refuses_scales_addresses_and_grids(kw, said):
    assert _attend(**dict(dict(nbytes=1 << 62), **kw)) == _C.ERR_ARG
    assert said.encode() in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


def test_eviction_needs_nothing_for_a_budget_that_no_sequence_reaches():
    need = _C.lib().mi355_kv_evict_workspace_bytes
    assert need(4, 8, 1 << 30, 4096) == need(4, 8, 4096, 4096) < 1 << 16
    assert _evict(M=1 << 26, most=(1 << 28) - 16) == _C.ERR_ARG and b"2^32" in _C.lib().mi355_last_error()


def test_attention_refuses_a_short_workspace():
    assert _C.lib().mi355_paged_attn_scored_workspace_bytes(1, 1, 1, 28, 4, 128, 64, 1) > 0
    assert _attend(weights=16, nbytes=0) == _C.ERR_WORKSPACE and _attend(weights=16, ws=None) == _C.ERR_WORKSPACE


def _evict(kv=None, *, w=16, pos=16, table=16, M=4, lens=16, nxt=16, B=1, most=64, keep=32, sinks=4, recent=8, ws=16, nbytes=1 << 30):
    return _C.lib().mi355_kv_evict(C.byref(kv or _kv()), w, pos, table, M, lens, nxt, B, most, keep, sinks, recent, None, ws, nbytes, None)


@pytest.mark.parametrize("kw,said", [(dict(w=None), "null"), (dict(pos=None), "null"), (dict(nxt=None), "null"), (dict(keep=0), "keep=0"), (dict(keep=11), "keep=11"), (dict(sinks=-1), "keep"),
                                     (dict(recent=(1 << 31) - 1), "keep"), (dict(most=65), "block table"), (dict(kv=_kv(hd=32)), "hd=32"), (dict(kv=_kv(page=8)), "page=8"), (dict(B=1 << 16), "B="),
                                     (dict(kv=_kv(kv_dtype=_C.KV_INT8, scale_base=None)), "scale"), (dict(kv=_kv(kv_base=24)), "16 bytes")])
def test_eviction_refuses(kw, said):
    assert _evict(**kw) == _C.ERR_ARG
    assert said.encode() in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


def test_eviction_refuses_a_short_workspace():
    need = _C.lib().mi355_kv_evict_workspace_bytes(1, 4, 32, 64)
    assert need > 0 and _evict(nbytes=need - 1) == _C.ERR_WORKSPACE and _evict(ws=None) == _C.ERR_WORKSPACE


def _write(kv=None, *, qkv=16, cs=16, slots=16, seq=None, B=1, T=1, q_len=1, nh=28, ld=36 * 128, M=4):
    return _C.lib().mi355_rope_kv_write_slots(qkv, ld, None, cs, 64, 16, slots, seq, 16, M, B, T, q_len, nh, C.byref(kv or _kv()), 16, None, None, None, None)


@pytest.mark.parametrize("kw,said", [(dict(qkv=None), "null"), (dict(slots=None), "null"), (dict(T=2), "2 rows"), (dict(seq=16, q_len=2, T=2), "q_len=2"), (dict(kv=_kv(hd=32)), "hd=32"),
                                     (dict(ld=100), "ld=100"), (dict(M=1 << 28), "blocks")])
def test_writer_refuses(kw, said):
    assert _write(**kw) == _C.ERR_ARG
    assert said.encode() in _C.lib().mi355_last_error(), _C.lib().mi355_last_error()


def test_ops_refuse_cpu_tensors():
    q, kv = torch.zeros(1, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 2, 16, 64, dtype=torch.float16)
    bt, one = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    w, pos = kvcache.alloc_planes(4, 2, 16, "cpu")
    with pytest.raises(_C.Mi355Error):
        ops.paged_attention_scored(q, kv, None, bt, one, 2, 16, 64)
    with pytest.raises(_C.Mi355Error):
        ops.kv_evict(w, pos, bt, one, one, kv, None, 16)
    with pytest.raises(_C.Mi355Error):
        ops.rope_kv_write_slots(torch.zeros(1, 512, dtype=torch.float16), None, None, one, one, bt, kv, None, 4, 2, 64, 16)


def test_the_oracle_of_moves():
    """Properties of the definition itself: sources and holes are disjoint and as many, what stays is the best, equal weights go to the lower slot."""
    rng = random.Random(1)
    for _ in range(200):
        n, keep = rng.randint(0, 60), rng.randint(1, 40)
        sinks = rng.randint(0, keep)
        recent = rng.randint(0, keep - sinks)
        w = [rng.choice([0.0, 1.0, rng.random()]) for _ in range(n)]
        pos = rng.sample(range(200), n)
        moves = evict(w, pos, n, keep, 200, sinks, recent)
        stay = [t for t in range(min(keep, n)) if t not in {d for _, d in moves}] + [s for s, _ in moves]
        assert len(stay) == min(n, keep) and all(s >= keep > d for s, d in moves) and moves == sorted(moves)
        safe = lambda t: pos[t] < sinks or pos[t] >= 200 - recent
        gone = set(range(n)) - set(stay)
        assert not any(safe(t) for t in gone)
        assert all(safe(s) or (w[s], -s) > (w[t], -t) for t in gone for s in stay)
