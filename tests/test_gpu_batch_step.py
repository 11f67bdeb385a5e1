"""GPU tests of a ragged serving step as it is used: the plan from lengths, the writes, and the
attention with a layer's score variant, masks and shared prefixes, through PagedKVPools and
paged_attention_step, against float64 attention over the dequantized rows (sequence_kv).

Tolerances, relative to the largest |value row|: 2e-5 for float32 queries (operands held to
2^-22, sums in fp32: see test_gpu_batch_attn.py) plus the 2^-22 that sequence_kv's own rows
are off; bfloat16: 1e-2 (2^-11 per operand, 2^-9 for the result)."""

import math

import numpy as np
import pytest
import torch

from turboquant_kv import TurboQuantConfig, ops
from turboquant_kv.vllm_plugin import (AttentionVariant, PagedKVPools, TurboQuantAttentionMetadata,
                                       TurboQuantKVCacheConfig, TurboQuantPagedKVCache, attention_variant,
                                       paged_attention_step)

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 2.2e-5, torch.float16: 2.2e-5 + 2.0 ** -11, torch.bfloat16: 1e-2}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def reference(pools, layer, q, md, variant, scale):
    qsl, lens = md.query_start_loc.tolist(), md.seq_lens.tolist()
    Hq = q.shape[1]
    G = Hq // pools.num_kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    size = torch.ones(q.shape[0], dtype=torch.float64, device=DEV)
    v = variant or AttentionVariant()
    for b, T in enumerate(lens):
        n = qsl[b + 1] - qsl[b]
        if n == 0 or T == 0:
            continue
        k, val = (x.double() for x in pools.sequence_kv(layer, md.block_tables[b], T))
        p = torch.arange(T - n, T, device=DEV)[:, None]
        j = torch.arange(T, device=DEV)[None]
        see = j <= p
        if md.prefix_lens is not None:
            see = see | (j < int(md.prefix_lens[b]))
        if v.window:
            see = see & (j > p - v.window)
        if md.token_starts is not None:
            see = see & (j >= md.token_starts[qsl[b]:qsl[b + 1], None])
        rows = q[qsl[b]:qsl[b + 1]].double()
        for h in range(Hq):
            x = rows[:, h] @ k[h // G].t() * scale
            if v.softcap:
                x = v.softcap * torch.tanh(x / v.softcap)
            if v.alibi_slopes is not None:
                x = x + float(v.alibi_slopes[h]) * (j - p)
            w = torch.softmax(x.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
            out[qsl[b]:qsl[b + 1], h] = w @ val[h // G]
        size[qsl[b]:qsl[b + 1]] = val.norm(dim=-1).max()
    return out, size


def check(got, ref, dtype):
    out, size = ref
    err = ((got.double() - out).norm(dim=-1).amax(-1) / size).max().item()
    assert err <= TOL[dtype], err


def _kv(rs, n, H, d, dtype):
    return (torch.from_numpy(rs.randn(n, H, d)).to(DEV).to(dtype) for _ in range(2))


def _q(rs, n, Hq, d, dtype):
    return torch.from_numpy(rs.randn(n, Hq, d)).to(DEV).to(dtype)


VARIANTS = [None, AttentionVariant(softcap=5.0), AttentionVariant(window=20),
            AttentionVariant(softcap=20.0, alibi_slopes=torch.tensor([2.0 ** -(i + 1) for i in range(8)]), window=60)]


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout,d,vb", [("decode", 64, 2), ("decode", 64, 4), ("bitplane", 64, 2), ("bitplane", 128, 3)])
def test_steps_from_lengths(layout, d, vb, dtype, variant):
    """Three steps (prompts, a mixed one, single tokens) of four requests whose blocks come from
    a free list, every step planned on the device."""
    rs = np.random.RandomState(3)
    pools = PagedKVPools(TurboQuantConfig(value_bits=vb), 1, 64, 16, 2, d, layout=layout)
    tables = torch.full((4, 12), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(1)).to(DEV, torch.int32)
    start = _ints([0])
    held = torch.zeros(4, dtype=torch.int32, device=DEV)
    for new, pad in (([30, 1, 70, 5], 0), ([1, 40, 0, 3], 3), ([1, 1, 1, 1], 1)):
        n = sum(new) + pad
        md, pos, used = TurboQuantAttentionMetadata.from_lengths(_ints(new), held, tables, free, 16, n, start)
        q, (k, v) = _q(rs, n, 8, d, dtype), _kv(rs, n, 2, d, dtype)
        got = pools.forward(q, k, v, md, 1 / math.sqrt(d), variant=variant)
        check(got, reference(pools, 0, q, md, variant, 1 / math.sqrt(d)), dtype)
        assert not got[sum(new):].any()
        held, start = md.seq_lens, start + used
    assert len(set(tables[tables >= 0].tolist())) == int((tables >= 0).sum())


@pytest.mark.parametrize("variant", [None, AttentionVariant(softcap=10.0, window=100)])
def test_shared_prompt(variant):
    """Requests behind one prompt: its blocks written once, found by their tables, attended once;
    masks of the metadata; protected layers beside packed ones."""
    rs = np.random.RandomState(5)
    cache = TurboQuantPagedKVCache(TurboQuantKVCacheConfig(num_gpu_blocks=80, value_bits=3, protected_layers=1), 2, 2, 64)
    pools = cache.pools()
    tables = torch.full((5, 16), -1, dtype=torch.int32, device=DEV)
    free = torch.arange(79, -1, -1, dtype=torch.int32, device=DEV)
    first, _, used = TurboQuantAttentionMetadata.from_lengths(_ints([96]), _ints([0]), tables[:1], free, 16, 96)
    for layer in range(2):
        k, v = _kv(rs, 96, 2, 64, torch.bfloat16)
        pools.write(layer, k, v, first.slot_mapping)
    tables[1:, :6] = tables[0, :6]
    held, new = _ints([96] * 5), [3, 1, 20, 1, 2]
    md, _, used2 = TurboQuantAttentionMetadata.from_lengths(_ints(new), held, tables, free, 16, 30, used,
                                                            min_shared_tokens=32)
    assert md.group_start_loc.tolist() == [0, 5, 5, 5, 5, 5] and md.shared_lens.tolist() == [96, 0, 0, 0, 0]
    md.prefix_lens = _ints([0, 97, 110, 50, 0])
    starts = torch.zeros(30, dtype=torch.int32, device=DEV)
    starts[4:8] = 90
    md.token_starts = starts
    for layer in range(2):
        md.layer_id = layer
        q, (k, v) = _q(rs, 30, 8, 64, torch.bfloat16), _kv(rs, 30, 2, 64, torch.bfloat16)
        out = torch.full((30, 8, 64), 3.0, dtype=torch.bfloat16, device=DEV)
        got = paged_attention_step(q, k, v, cache, md, 0.125, out, variant)
        assert got is out and bool((out[27:] == 3).all())
        ref = reference(pools, layer, q, md, variant, 0.125)
        check(out[:27], (ref[0][:27], ref[1][:27]), torch.bfloat16)
        alone = paged_attention_step(q, k, v, cache, md, 0.125, None, variant)
        assert torch.equal(alone[:27], out[:27]) and not alone[27:].any()


def test_result_in_the_queries_memory():
    rs = np.random.RandomState(6)
    pools = PagedKVPools(TurboQuantConfig(), 1, 16, 16, 2, 64, layout="decode")
    tables = torch.arange(16, dtype=torch.int32, device=DEV).view(2, 8)
    free = torch.arange(0, dtype=torch.int32, device=DEV)
    k, v = _kv(rs, 60, 2, 64, torch.bfloat16)
    t = torch.arange(60, device=DEV)
    pools.write(0, k, v, torch.where(t < 40, t, 128 + t - 40))
    md = TurboQuantAttentionMetadata(None, _ints([40, 20]), tables, _ints([0, 4, 5]), 0, ragged=True)
    q = _q(rs, 6, 8, 64, torch.bfloat16)
    want = pools.attend(0, q, md, 0.125)
    same = q.clone()
    pools.attend(0, same, md, 0.125, output=same)
    assert torch.equal(same[:5], want[:5]) and torch.equal(same[5:], q[5:])
    other = torch.zeros(6, 8, 64, device=DEV)  # another type
    pools.attend(0, q, md, 0.125, output=other)
    assert torch.equal(other[:5], want[:5].float())
    assert pools.attend(0, q.double(), md, 0.125).dtype == torch.float64


def test_impl_arguments():
    v = attention_variant([0.5, 0.25], 128, 30.0)
    assert v.softcap == 30.0 and v.window == 128 and v.alibi_slopes.tolist() == [0.5, 0.25] and bool(v)
    assert not attention_variant(None, None, None) and not attention_variant(None, -1, 0.0)


def test_step_captured_and_replayed():
    """A whole layer's step -- plan, groups, writes, attention -- in a graph, replayed as the
    requests grow, against the eager step on a copy of the state."""
    rs = np.random.RandomState(7)
    dt = torch.bfloat16
    pools = [PagedKVPools(TurboQuantConfig(value_bits=2), 1, 40, 16, 2, 64, layout="decode") for _ in range(2)]
    tables = [torch.full((3, 8), -1, dtype=torch.int32, device=DEV) for _ in range(2)]
    free = torch.arange(40, dtype=torch.int32, device=DEV)
    new, n = _ints([1, 1, 1]), 4
    held, start = _ints([0, 0, 0]), _ints([0])
    q, (k, v) = _q(rs, n, 8, 64, dt), _kv(rs, n, 2, 64, dt)
    variant = AttentionVariant(softcap=20.0, alibi_slopes=torch.tensor([0.1] * 8))

    def step(i):
        md, _, used = TurboQuantAttentionMetadata.from_lengths(new, held, tables[i], free, 16, n, start,
                                                               min_shared_tokens=16)
        return pools[i].forward(q, k, v, md, 0.125, variant=variant), md.seq_lens, used

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lens, used = step(0)
    for t in range(40):
        q.copy_(_q(rs, n, 8, 64, dt)), k.copy_(next(_kv(rs, n, 2, 64, dt))), v.copy_(next(_kv(rs, n, 2, 64, dt)))
        graph.replay()
        want, lens2, used2 = step(1)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lens, lens2) and torch.equal(tables[0], tables[1])
        held.copy_(lens2), start.add_(used2)
    assert held.tolist() == [40, 40, 40] and start.item() == 9
    check(out[:3], tuple(x[:3] for x in reference(pools[1], 0, q, TurboQuantAttentionMetadata(
        None, held, tables[1], _ints([0, 1, 2, 3]), 0), variant, 0.125)), dt)
