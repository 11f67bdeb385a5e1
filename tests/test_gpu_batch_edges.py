"""GPU tests of the ragged batch's attention at its limits: pools past 4 GB, most sequences, long
contexts in many pieces, rows of very different sizes, odd head counts, masks of 64 bits.

Tolerances are those of test_gpu_batch_attn.py, per row, relative to its largest visible value; a
result that the same arithmetic must give is compared bit by bit.
"""

import math

import numpy as np
import pytest
import torch

from test_gpu_batch_attn import DEV, DTYPES, Pools, _ints, _tables, check, run, want
from turboquant_kv import TurboQuantConfig, ops
from turboquant_kv.vllm_plugin import AttentionVariant, PagedKVPools, TurboQuantAttentionMetadata

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs,vb,H,nblocks", [(64, 4, 2, 2 ** 20 - 1), (64, 4, 2, 2 ** 20 + 5), (16, 3, 1, 2 ** 23 - 1),
                                             (16, 3, 1, 2 ** 23 + 3), (16, 2, 1, 2 ** 23 + 3), (32, 4, 2, 2 ** 21 + 1),
                                             (64, 3, 2, 2 ** 20 + 1)])
def test_pools_past_4gb(bs, vb, H, nblocks):
    """Key bytes just below 2^32 and past it: the blocks lie at both ends and in the middle, and
    the results are those of a small pool of the same blocks."""
    rs = np.random.RandomState(30)
    n = 40
    P = Pools(21, n, H, bs, vb)
    ids = np.concatenate([[nblocks - 1, 0, nblocks // 2], rs.choice(np.arange(1, nblocks // 2 - 1), n - 3, replace=False)])
    ids[3::2] = nblocks - 1 - ids[3::2]
    at = torch.from_numpy(ids.astype(np.int64)).to(DEV)
    big = []
    for small in P.args():
        t = torch.empty(nblocks, *small.shape[1:], dtype=small.dtype, device=DEV)
        t[at] = small
        big.append(t)
    assert (big[0].numel() > 2 ** 32) == (nblocks % 16 < 8)
    lens = [3 * bs + 5, 9 * bs, 2 * bs + 1, 7 * bs - 1]
    tab = _tables(rs, lens, bs, n, fill=0)
    tab[1, :2] = tab[0, :2]
    for new in ([1, 1, 1, 1], [2, 9 * bs, 1, 40]):
        q = torch.from_numpy(rs.randn(sum(new), 4 * H, 64)).to(DEV)
        at_q = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(DEV)
        for dt in ("f32", "bf16"):
            for fn, extra in ((ops.attention_batch_paged_dl, ()),
                              (ops.attention_shared_prefix_paged_dl, (_ints([0, 2]), _ints([2 * bs])))):
                got = [fn(q.to(DTYPES[dt]), *pools, torch.from_numpy(t).to(DEV), at_q, _ints(lens), *extra, *P.tables(), 0.125)
                       for pools, t in ((P.args(), tab), (big, ids[tab].astype(np.int32)))]
                assert torch.equal(*got), (new, dt, bool(extra))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,new,T", [(8, [1], 70000), (8, [1, 1, 1], 30000), (40, [1], 40000), (8, [9], 40000),
                                      (8, [70, 1], 20000), (16, [1, 1], 33333)])
def test_one_head_in_many_pieces(dt, Hq, new, T):
    """Few rows over a long context of one KV head: hundreds of pieces to join."""
    rs = np.random.RandomState(31)
    P = Pools(22, 1100, 1, 64, 2)
    run(P, rs, new, [T] + [65 * i for i in range(1, len(new))], Hq, dt)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,Hq", [(8, 8), (32, 32), (1, 40), (2, 64), (1, 128), (5, 35)])
def test_many_heads(dt, H, Hq):
    rs = np.random.RandomState(32)
    P = Pools(23, 60, H, 16, 2)
    run(P, rs, [1, 1, 3], [200, 17, 300], Hq, dt)
    run(P, rs, [40, 1], [45, 600], Hq, dt, pad=1)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [[1, 1], [30, 2]])
def test_queries_of_very_different_sizes(dt, new):
    """Rows of one wave share a power of two: heads 2^-14 shorter than others, and zeros (whose
    weights are equal).  16-bit floats hold these queries as normal numbers, but for f16's tail,
    which is part of the query that the definition gets."""
    rs = np.random.RandomState(33)
    P = Pools(24, 60, 2, 16, 2)
    lens = [300, 170]
    tab = _tables(rs, lens, 16, P.nb)
    q = torch.from_numpy(rs.randn(sum(new), 8, 64)).to(DEV)
    q *= torch.tensor([1.0, 2.0 ** -14, 0.0, 2.0 ** -7, 2.0 ** -3, 1.0, 2.0 ** -10, 0.0], device=DEV)[:, None]
    q = q.to(DTYPES[dt])
    at = _ints([0, new[0], sum(new)])
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), torch.from_numpy(tab).to(DEV), at, _ints(lens), *P.tables(), 0.125,
                                            return_lse=True)
    check(got, lse, want(P, q, tab, new, lens, 0.125), dt)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [[1, 1], [30, 2]])
def test_a_bad_query_spoils_its_own_rows_only(new, bad):
    rs = np.random.RandomState(34)
    P = Pools(25, 60, 2, 16, 2)
    lens = [300, 170]
    tab = _tables(rs, lens, 16, P.nb)
    for dt in ("f32", "bf16"):
        q = torch.from_numpy(rs.randn(sum(new), 8, 64)).to(DEV).to(DTYPES[dt])
        spoilt = q.clone()
        spoilt[0, 1, 5] = bad
        at = _ints([0, new[0], sum(new)])
        got, lse = ops.attention_batch_paged_dl(spoilt, *P.args(), torch.from_numpy(tab).to(DEV), at, _ints(lens),
                                                *P.tables(), 0.125, return_lse=True)
        ref = want(P, q, tab, new, lens, 0.125)
        assert bool(got[0, 1].isnan().all())
        keep = torch.ones(sum(new), 8, dtype=torch.bool, device=DEV)
        keep[0, 1] = False
        check(got[keep], lse[keep], tuple(x[keep] for x in ref), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("down", [2.0 ** -60, 2.0 ** 60])
def test_very_small_and_large_values(dt, down):
    """Value norms far outside fp16's range: results scale with them (powers of two: exactly)."""
    rs = np.random.RandomState(35)
    P = Pools(26, 60, 2, 16, 2)
    lens, new = [300, 170, 64], [1, 2, 1]
    t = torch.from_numpy(_tables(rs, lens, 16, P.nb)).to(DEV)
    q = torch.from_numpy(rs.randn(4, 8, 64)).to(DEV).float()
    a = (t, _ints([0, 1, 3, 4]), _ints(lens), *P.tables(), 0.125)
    got = ops.attention_batch_paged_dl(q, P.kp, P.kn, P.vt, P.vn, *a)
    far = ops.attention_batch_paged_dl(q, P.kp, P.kn, P.vt, P.vn * down, *a)
    assert torch.allclose(far.double() / down, got.double(), rtol=0, atol=2e-5 * P.vn.max().item())


def test_most_sequences():
    rs = np.random.RandomState(36)
    P = Pools(27, 64, 1, 16, 2)
    B = 8192
    tab = rs.randint(0, 64, (B, 2)).astype(np.int32)
    lens = rs.randint(0, 33, B)
    q = torch.from_numpy(rs.randn(B, 2, 64)).to(DEV).float()
    at, sl, t = torch.arange(B + 1, dtype=torch.int32, device=DEV), torch.from_numpy(lens).to(DEV), torch.from_numpy(tab).to(DEV)
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), t, at, sl, *P.tables(), 0.125, return_lse=True)
    some = np.concatenate([np.arange(0, B, 331), [B - 2, B - 1]])
    i = torch.from_numpy(some).to(DEV)
    check(got[i], lse[i], want(P, q[i], tab[some], [1] * len(some), lens[some].tolist(), 0.125), "f32")
    groups, shared = ops.shared_prefix_groups(t, sl, 16, 16)
    both = ops.attention_shared_prefix_paged_dl(q, *P.args(), t, at, sl, groups, shared, *P.tables(), 0.125)
    check(both[i], None, want(P, q[i], tab[some], [1] * len(some), lens[some].tolist(), 0.125), "f32")
    with pytest.raises(RuntimeError, match="8192"):
        ops.attention_batch_paged_dl(q, *P.args(), torch.zeros(B + 1, 1, dtype=torch.int32, device=DEV),
                                     torch.zeros(B + 2, dtype=torch.int32, device=DEV),
                                     torch.zeros(B + 1, dtype=torch.int32, device=DEV), *P.tables(), 0.125)


def test_one_table_twice_and_result_in_the_queries():
    """Two sequences over the same blocks; a result written over the queries, or over part of
    them, is the one written elsewhere."""
    rs = np.random.RandomState(37)
    P = Pools(28, 60, 2, 16, 2)
    for new in ([1, 1, 1], [50, 50, 3]):
        lens, n = [300, 300, 90], sum(new)
        tab = _tables(rs, lens, 16, P.nb)
        tab[1] = tab[0]
        x = torch.from_numpy(rs.randn(n + 4, 8, 64)).to(DEV).bfloat16()
        x[new[0]:2 * new[0]] = x[:new[0]]
        a = (torch.from_numpy(tab).to(DEV), _ints([0, new[0], 2 * new[0], n]), _ints(lens), *P.tables(), 0.125)
        ref = ops.attention_batch_paged_dl(x[:n], *P.args(), *a)
        assert torch.equal(ref[:new[0]], ref[new[0]:2 * new[0]])
        for shift in (0, 3):
            y = x.clone()
            ops.attention_batch_paged_dl(y[:n], *P.args(), *a, out=y[shift:shift + n])
            assert torch.equal(y[shift:shift + n], ref)


def test_masks_of_64_bits():
    """Starts and prefixes past 32 bits mean what they say: nothing, or everything, is visible."""
    rs = np.random.RandomState(38)
    P = Pools(29, 60, 2, 16, 2)
    lens, new = [100, 60], [3, 1]
    tab = _tables(rs, lens, 16, P.nb)
    q = torch.from_numpy(rs.randn(4, 8, 64)).to(DEV).float()
    a = (torch.from_numpy(tab).to(DEV), _ints([0, 3, 4]), _ints(lens), *P.tables(), 0.125)
    starts = torch.tensor([2 ** 63 - 1, 2 ** 33, -2 ** 40, 0], device=DEV)
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), *a, token_starts=starts, return_lse=True)
    check(got, lse, want(P, q, tab, new, lens, 0.125, starts=starts.tolist()), "f32")
    prefix = torch.tensor([2 ** 40, -2 ** 63], device=DEV)
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), *a, prefix_lens=prefix, return_lse=True)
    check(got, lse, want(P, q, tab, new, lens, 0.125, prefix=prefix.tolist()), "f32")


def test_two_graphs_in_turn():
    """Two captured calls keep their own workspaces: replayed in turn, each gives its eager result."""
    rs = np.random.RandomState(39)
    P = Pools(30, 120, 2, 16, 2)
    t = torch.from_numpy(_tables(rs, [300, 280], 16, P.nb)).to(DEV)
    sl = _ints([300, 280])
    qs, graphs, outs = [], [], []
    for new in (1, 60):
        q = torch.from_numpy(rs.randn(2 * new, 8, 64)).to(DEV).bfloat16()
        at = _ints([0, new, 2 * new])
        call = lambda q=q, at=at: ops.attention_batch_paged_dl(q, *P.args(), t, at, sl, *P.tables(), 0.125)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        qs.append((q, call))
        graphs.append(g)
    for step in range(3):
        sl.copy_(_ints([300 - 7 * step, 80 + 100 * step]))
        for g, (q, _) in zip(graphs, qs):
            q.copy_(torch.from_numpy(rs.randn(*q.shape)))
            g.replay()
        torch.cuda.synchronize()
        for out, (_, call) in zip(outs, qs):
            assert torch.equal(out, call())


@pytest.mark.parametrize("softcap", [1e-40, 1e-31, 1e31, 3e38, -0.5, math.nan])
def test_softcaps_out_of_range(softcap):
    P = Pools(31, 4, 2, 16, 2)
    q = torch.randn(1, 8, 64, device=DEV)
    with pytest.raises(RuntimeError, match="softcap"):
        ops.attention_batch_paged_dl(q, *P.args(), torch.zeros(1, 2, dtype=torch.int32, device=DEV), _ints([0, 1]), _ints([9]),
                                     *P.tables(), 0.125, softcap=softcap)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1], [30, 2]])
def test_subnormal_queries_and_values(dt, new):
    """Queries and value norms near the end of fp32: weights are equal to rounding, and results are
    as small as the values, whose rows of about 2^-114 an fp32 subnormal's 2^-149 resolves to 2^-35."""
    rs = np.random.RandomState(40)
    P = Pools(32, 60, 2, 16, 2)
    lens = [300, 170]
    tab = _tables(rs, lens, 16, P.nb)
    q = (torch.from_numpy(rs.randn(sum(new), 8, 64)).to(DEV) * 2.0 ** -122).to(DTYPES[dt])
    small = P.vn * 2.0 ** -115
    a = (torch.from_numpy(tab).to(DEV), _ints([0, new[0], sum(new)]), _ints(lens), *P.tables(), 0.125)
    got, lse = ops.attention_batch_paged_dl(q, P.kp, P.kn, P.vt, small, *a, return_lse=True)
    out, wl, size = want(P, q, tab, new, lens, 0.125)
    check(got.double() * 2.0 ** 115, lse, (out, wl, size), dt)


@pytest.mark.parametrize("inference", [False, True])
def test_small_results_are_tensors_of_their_own(inference):
    """A plan's and the groups' results come from one allocation each: writing one leaves the others,
    with and without inference mode, and each outlives the rest."""
    with torch.inference_mode(inference):
        tab = torch.zeros(3, 4, dtype=torch.int32, device=DEV)
        args = (_ints([2, 0, 5]), _ints([0, 16, 3]), tab, torch.arange(10, 20, dtype=torch.int32, device=DEV), 16, 9)
        first = ops.paged_batch_plan(*args)
        kept = [x.clone() for x in first]
        assert [x.numel() for x in first] == [4, 3, 9, 9, 9, 1] and all(x.is_contiguous() for x in first)
        for i, x in enumerate(first):
            x.fill_(-9)
            for y, z in zip(first[i + 1:], kept[i + 1:]):
                assert torch.equal(y, z)
        used = ops.paged_batch_plan(_ints([2, 0, 5]), _ints([0, 16, 3]), tab, args[3], 16, 9)[5]
        torch.empty(1 << 20, device=DEV).fill_(7.0)
        assert used.tolist() == [1]
        same = torch.ones(3, 4, dtype=torch.int32, device=DEV)
        starts, shared = ops.shared_prefix_groups(same, _ints([64, 64, 64]), 16, 16)
        starts.fill_(5)
        assert shared.tolist() == [64, 0, 0]


@pytest.mark.parametrize("layout", ["decode", "bitplane"])
def test_steps_without_starts_and_on_the_host(layout):
    """A decode step's metadata without query_start_loc means a token per sequence; queries and a
    result on the host give what the device gives."""
    g = torch.Generator(device=DEV).manual_seed(41)
    pools = PagedKVPools(TurboQuantConfig(), 1, 8, 16, 2, 64, layout=layout)
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    k, v = (torch.randn(100, 2, 64, device=DEV, generator=g) for _ in range(2))
    t = torch.arange(100, device=DEV)
    pools.write(0, k, v, torch.where(t < 60, t, 64 + t - 60))
    q = torch.randn(2, 8, 64, device=DEV, generator=g)
    variant = AttentionVariant(softcap=20.0, window=50)
    with_starts = TurboQuantAttentionMetadata(None, _ints([60, 40]), tables, _ints([0, 1, 2]), 0)
    without = TurboQuantAttentionMetadata(None, _ints([60, 40]), tables, None, 0)
    ref = pools.attend(0, q, with_starts, 0.125, variant)
    assert torch.equal(pools.attend(0, q, without, 0.125, variant), ref)
    host = pools.attend(0, q.cpu(), without, 0.125, variant)
    assert host.device.type == "cpu" and torch.equal(host, ref.cpu())
    dst = torch.full((2, 8, 64), 3.0)
    assert pools.attend(0, q, without, 0.125, variant, dst) is dst and torch.equal(dst, ref.cpu())
