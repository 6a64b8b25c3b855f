"""What the scored decode implementation hands to its operators, on the host: the bound on slots, the rotation, the planes."""
import pytest
import torch

from rtp_llm_amd import kvcache
from rtp_llm_amd import attention as A

NH, NKV, HD, PAGE = 8, 2, 64, 16


def impl_of(monkeypatch, calls, *, table_blocks, lens, positions=None, cos_sin=None, graph=False, **cfg):
    """An implementation whose operators only note their arguments."""
    def write(qkv, bias, cos, pos, slots, *a, **kw):
        calls.append(("write", cos, pos.clone(), slots.clone(), kw))
        return qkv.view(qkv.shape[0], -1, HD)[:, :NH]

    def attend(q, kv, sc, bt, end, nkv, page, most, **kw):
        calls.append(("attend", most, end.clone(), kw))
        return q.reshape(q.shape[0], -1)

    def evict(w, pos, bt, lens, nxt, kv, sc, keep, **kw):
        calls.append(("evict", bt.shape[1] * PAGE if kw.get("max_seq_len") is None else kw["max_seq_len"], lens.clone(), nxt.clone(), keep))
        return lens.clamp(max=keep)

    for name, f in (("rope_kv_write_slots", write), ("paged_attention_scored", attend), ("kv_evict", evict)):
        monkeypatch.setattr(A.ops, name, f)
    inputs = A.PyAttentionInputs(sequence_lengths=lens, kv_cache_kernel_block_id_device=torch.zeros(len(lens), table_blocks, dtype=torch.int32), token_positions=positions,
                                is_cuda_graph=graph)
    return A.AttnImplFactory.get_fmha_impl(A.AttentionConfigs(NH, NKV, HD, **cfg), inputs, cos_sin=cos_sin)


def cache(planes=True):
    w, pos = kvcache.alloc_planes(8, NKV, PAGE, "cpu") if planes else (None, None)
    return A.LayerKVCache(torch.zeros(8, 2, NKV, PAGE, HD, dtype=torch.float16), None, PAGE, 0, w, pos)


@pytest.mark.parametrize("table_blocks,max_seq_len", [(3, 4096), (300, 4096)])
def test_slots_are_bounded_by_the_table(monkeypatch, table_blocks, max_seq_len):
    """max_seq_len bounds positions.  A budget's table may be shorter, and a longer one's slots are all written, attended and ranked."""
    calls = []
    impl = impl_of(monkeypatch, calls, table_blocks=table_blocks, lens=torch.tensor([30, 47]), positions=torch.tensor([2000, 4000]), cos_sin=torch.zeros(4096, HD // 2, 2), rope_dim=HD,
                   max_seq_len=max_seq_len, kv_budget=32, kv_sinks=2, kv_recent=8)
    impl.forward(torch.zeros(2, (NH + 2 * NKV) * HD, dtype=torch.float16), cache())
    impl.evict(cache())
    (_, _, pos, slots, _), (_, most, end, _), (_, ranked, lens, nxt, keep) = calls
    assert most == ranked == table_blocks * PAGE
    assert slots.tolist() == [30, 47] and pos.tolist() == [2000, 4000] and end.tolist() == lens.tolist() == [31, 48] and nxt.tolist() == [2001, 4001] and keep == 32


def test_rotated_models_need_the_rotation(monkeypatch):
    """No table means no rotation to the writer: a model that rotates is refused without one, one with slopes or without rotated channels runs."""
    table, lens = torch.zeros(64, HD // 2, 2), torch.tensor([3])
    for cfg in (dict(softcap=30.0), dict(kv_budget=40), dict(softcap=30.0, kv_budget=40)):
        with pytest.raises(ValueError, match="cos_sin"):
            impl_of(monkeypatch, [], table_blocks=4, lens=lens, rope_dim=HD, **cfg)
        calls = []
        impl_of(monkeypatch, calls, table_blocks=4, lens=lens, rope_dim=HD, cos_sin=table, **cfg).forward(torch.zeros(1, (NH + 2 * NKV) * HD, dtype=torch.float16), cache())
        assert calls[0][1] is table
    for cfg in (dict(slopes=torch.ones(NH), rope_dim=HD), dict(softcap=30.0, rope_dim=0), dict(slopes=torch.ones(NH), rope_dim=0)):
        calls = []
        impl_of(monkeypatch, calls, table_blocks=4, lens=lens, **cfg).forward(torch.zeros(1, (NH + 2 * NKV) * HD, dtype=torch.float16), cache())
        assert calls[0][1] is None


def test_eviction_needs_planes_and_a_budget(monkeypatch):
    lens = torch.tensor([3])
    impl = impl_of(monkeypatch, [], table_blocks=4, lens=lens, kv_budget=40)
    with pytest.raises(ValueError, match="planes"):
        impl.evict(cache(planes=False))
    impl = impl_of(monkeypatch, [], table_blocks=4, lens=lens, softcap=30.0)
    with pytest.raises(ValueError, match="budget"):
        impl.evict(cache())


@pytest.mark.parametrize("cfg,said", [(dict(softcap=-30.0), "softcap"), (dict(kv_budget=-1), "kv_budget"), (dict(softcap=float("nan")), "softcap"), (dict(softcap=30.0, kv_budget=-1), "kv_budget")])
def test_forms_that_are_none_are_refused(monkeypatch, cfg, said):
    """A cap or a budget below zero is no plain configuration: it is refused, not left out."""
    with pytest.raises(ValueError, match=said):
        impl_of(monkeypatch, [], table_blocks=4, lens=torch.tensor([3]), **cfg)


def test_refreshed_buffers_are_the_implementations_own(monkeypatch):
    """prepare_cuda_graph refreshes buffers in place: not the lengths, positions and tables that the first inputs came with."""
    calls = []
    lens, positions = torch.tensor([3, 5], dtype=torch.int32), torch.tensor([30, 50], dtype=torch.int32)
    impl = impl_of(monkeypatch, calls, table_blocks=4, lens=lens, positions=positions, graph=True, kv_budget=40)
    table = impl.inputs.kv_cache_kernel_block_id_device
    kept = [x.clone() for x in (lens, positions, table)]
    at = [x.data_ptr() for x in (impl.slots, impl.positions, impl.seq_lens, impl.block_table)]
    impl.prepare_cuda_graph(A.PyAttentionInputs(sequence_lengths=lens + 1, kv_cache_kernel_block_id_device=table + 7, token_positions=positions + 1))
    assert [x.data_ptr() for x in (impl.slots, impl.positions, impl.seq_lens, impl.block_table)] == at
    assert impl.slots.tolist() == [4, 6] and impl.positions.tolist() == [31, 51] and impl.seq_lens.tolist() == [5, 7] and bool((impl.block_table == 7).all())
    assert all(torch.equal(a, b) for a, b in zip((lens, positions, table), kept))
