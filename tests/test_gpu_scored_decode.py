"""Tracked writes, scored attention and eviction as they are used together: decode steps of a cache with a budget through the attention factory, against a model of the same in 64 bits that holds
every (sequence, head)'s tokens as a list."""
import pytest
import torch

from rtp_llm_amd import kvcache
from rtp_llm_amd.attention import AttentionConfigs, AttnImplFactory, LayerKVCache, Mi355PagedDecodeImpl, Mi355ScoredDecodeImpl, PyAttentionInputs
from tests.scored_util import U, evict

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,nh,nkv,hd,page,form", [(torch.float16, 8, 2, 64, 16, "cap"), (torch.bfloat16, 14, 2, 128, 32, "slopes"), (torch.float16, 28, 4, 128, 16, "plain")])
def test_steps_of_a_cache_with_a_budget(dtype, nh, nkv, hd, page, form):
    g = torch.Generator(device=DEV).manual_seed(nh)
    B, budget, steps, every = 3, 40, 72, 12
    c = AttentionConfigs(nh, nkv, hd, rope_dim=0 if form == "slopes" else hd, max_seq_len=96, kv_budget=budget, kv_sinks=2, kv_recent=8, kv_decay=0.95,
                         softcap=4.0 if form == "cap" else 0.0, slopes=torch.tensor([0.5 ** (1 + h / 4) for h in range(nh)], device=DEV) if form == "slopes" else None)
    ang = torch.arange(256, device=DEV, dtype=torch.float64)[:, None] * 0.7 ** torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float()
    M = -(-96 // page)
    kv, _ = kvcache.alloc_layer_cache(B * M + 1, nkv, page, hd, False, DEV, dtype)
    w, pos = kvcache.alloc_planes(B * M + 1, nkv, page, DEV)
    cache = LayerKVCache(kv, None, page, 0, w, pos)
    bt = torch.randperm(B * M + 1, generator=torch.Generator().manual_seed(1))[: B * M].reshape(B, M).int().to(DEV)
    lens = torch.tensor([0, 5, 0], dtype=torch.int32)[:B]
    positions = lens.clone()
    lens.zero_()
    model = [[dict(k=[], v=[], w=[], p=[]) for _ in range(nkv)] for _ in range(B)]        # a list position is a slot
    u, moved = U[dtype], 0
    for step in range(steps):
        inputs = PyAttentionInputs(sequence_lengths=lens, kv_cache_kernel_block_id_device=bt, token_positions=positions)
        impl = AttnImplFactory.get_fmha_impl(c, inputs, cos_sin=cs)
        assert type(impl) is Mi355ScoredDecodeImpl
        qkv = torch.randn(B, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(dtype)
        out = impl.forward(qkv, cache).view(B, nh, hd).double()
        x = qkv.view(B, nh + 2 * nkv, hd)
        for b in range(B):
            t = int(positions[b])
            rot = x[b].float()
            if form != "slopes":
                co, si = cs[t, :, 0], cs[t, :, 1]
                rot = torch.cat([co * rot[:, : hd // 2] - si * rot[:, hd // 2:], co * rot[:, hd // 2:] + si * rot[:, : hd // 2]], -1)
            rot = rot.to(dtype).double()
            for h in range(nkv):
                m = model[b][h]
                m["k"].append(rot[nh + h]); m["v"].append(x[b, nh + nkv + h].double()); m["w"].append(0.0); m["p"].append(t)
                K, V = torch.stack(m["k"]), torch.stack(m["v"])
                s = rot[h * (nh // nkv):(h + 1) * (nh // nkv)] @ K.t().contiguous() * hd ** -0.5
                if form == "cap":
                    s = 4.0 * torch.tanh(s / 4.0)
                if form == "slopes":
                    s = s + c.slopes[h * (nh // nkv):(h + 1) * (nh // nkv), None].double() * (torch.tensor(m["p"], device=DEV) - t)
                p = s.softmax(-1)
                want, size = p @ V, p @ V.abs()
                got = out[b, h * (nh // nkv):(h + 1) * (nh // nkv)]
                # a rotated key or query may round to the other neighbour where the fp32 rotation is next to a border: one step of one of hd products, of a score and so of a weight
                tol = u * (want.abs() + size) + (2 * u * 16 * hd ** -0.5 + 1e-4) * size
                assert bool(((got - want).abs() <= tol).all()), (step, b, h, float(((got - want).abs() / tol).max()))
                have = w[bt[b].long(), h].reshape(-1)[: len(m["w"])]
                ref = torch.tensor(m["w"], device=DEV, dtype=torch.float64) * 0.95 + p.sum(0)
                assert bool(((have.double() - ref).abs() <= 1e-4 + (2 * u * 16 * hd ** -0.5 + 1e-4) * ref).all()), (step, b, h)
                m["w"] = have.double().tolist()                                            # ranks go by the framework's own weights from here on
                assert pos[bt[b].long(), h].reshape(-1)[: len(m["p"])].tolist() == m["p"]
        lens, positions = lens + 1, positions + 1
        if step % every == every - 1:
            new = impl.evict(cache)
            for b in range(B):
                for h in range(nkv):
                    m, n = model[b][h], int(lens[b])
                    for src, hole in evict(m["w"], m["p"], n, budget, int(positions[b]), 2, 8):
                        moved += 1
                        for name in m:
                            m[name][hole] = m[name][src]
                    for name in m:
                        del m[name][budget:]
            assert new.tolist() == [min(int(n), budget) for n in lens]
            lens = new.cpu()
    assert moved > 100


@pytest.mark.parametrize("int8", [False, True])
def test_captured_steps(int8):
    """A step's write, attention and eviction in one graph, replayed step after step with eager work between: bit for bit the eager chain on a cache of its own."""
    dtype, nh, nkv, hd, page, B, budget = torch.float16, 16, 4, 128, 16, 3, 24
    c = AttentionConfigs(nh, nkv, hd, rope_dim=hd, max_seq_len=64, kv_budget=budget, kv_sinks=2, kv_recent=6, softcap=20.0)
    ang = torch.arange(128, device=DEV, dtype=torch.float64)[:, None] * 0.7 ** torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float()
    bt = torch.randperm(B * 4 + 1, generator=torch.Generator().manual_seed(2))[: B * 4].reshape(B, 4).int().to(DEV)
    g = torch.Generator(device=DEV).manual_seed(9)
    caches = []
    for _ in range(2):
        kv, sc = kvcache.alloc_layer_cache(B * 4 + 1, nkv, page, hd, int8, DEV, dtype)
        kv.zero_()
        if sc is not None:
            sc.zero_()
        caches.append(LayerKVCache(kv, sc, page, 0, *kvcache.alloc_planes(B * 4 + 1, nkv, page, DEV)))
    lens, positions = torch.tensor([0, 0, 0], dtype=torch.int32), torch.tensor([0, 3, 1], dtype=torch.int32)
    qkv = torch.zeros(B, (nh + 2 * nkv) * hd, device=DEV, dtype=dtype)
    inputs = lambda: PyAttentionInputs(sequence_lengths=lens, kv_cache_kernel_block_id_device=bt, token_positions=positions, is_cuda_graph=True)
    impl, gr = AttnImplFactory.get_fmha_impl(c, inputs(), cos_sin=cs), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):                                               # nothing runs here
        out = impl.forward(qkv, caches[0])
        new = impl.evict(caches[0])
    for step in range(60):
        qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=g))
        impl.prepare_cuda_graph(inputs())
        gr.replay()
        eager = AttnImplFactory.get_fmha_impl(c, inputs(), cos_sin=cs)
        want = eager.forward(qkv, caches[1])
        want_new = eager.evict(caches[1])
        assert torch.equal(out, want) and torch.equal(new, want_new) and new.tolist() == [min(step + 1, budget)] * B, step
        a, b = caches
        assert torch.equal(a.kv_cache_base, b.kv_cache_base) and torch.equal(a.weights, b.weights) and torch.equal(a.key_pos, b.key_pos), step
        assert not int8 or torch.equal(a.kv_scale_base, b.kv_scale_base)
        lens, positions = new.cpu(), positions + 1


def test_plain_configurations_keep_their_implementation():
    inputs = PyAttentionInputs(sequence_lengths=torch.tensor([3]), kv_cache_kernel_block_id_device=torch.zeros(1, 2, dtype=torch.int32, device=DEV))
    assert type(AttnImplFactory.get_fmha_impl(AttentionConfigs(8, 2, 64), inputs)) is Mi355PagedDecodeImpl
    assert type(AttnImplFactory.get_fmha_impl(AttentionConfigs(8, 2, 64, softcap=30.0), inputs)) is Mi355ScoredDecodeImpl
    with pytest.raises(ValueError):
        cache = LayerKVCache(torch.zeros(2, 2, 2, 16, 64, device=DEV, dtype=torch.float16), None, 16)
        AttnImplFactory.get_fmha_impl(AttentionConfigs(8, 2, 64, kv_budget=8), inputs).forward(torch.zeros(1, 12 * 64, device=DEV, dtype=torch.float16), cache)
