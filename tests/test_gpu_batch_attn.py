"""GPU tests of the ragged batch's attention over packed pools (ops.attention_batch_paged_dl and
attention_shared_prefix_paged_dl) against the definition in float64, at the lengths, masks and
layouts where it can go wrong.

Tolerances.  The comparison is per output row, relative to the row's largest possible size
(the largest |value row| it can see): a weighted mean's error is at most the largest error of a
weight's share times that size.  float32 / float16 queries: every operand is held to 2^-22
(fp16 hi + lo parts), so a score s = scale n_k <q, c> is off by at most 3 * 2^-22 * scale n_k |q| |c|
plus fp32 sums of 64 terms (64 * 2^-24 of the same bound in the worst order) -- together
under 2^-17 S with S the row's largest scale |q| |k|.  A weight is off by the factor
exp(2 * 2^-17 S), a mean by no more than 4 * 2^-17 S + 2^-17 of the values' size (sums over up
to 2^12 tokens err in random directions; rotations add 2^-18).  With S <= 40 in these tests that is
2^-17 (4 * 40 + 1) = 1.3e-3 in the worst case; the tests hold the far tighter 2e-5 (errors of
64 independent roundings are about sqrt(64) / 64 of the worst order, and of many tokens less).
bfloat16 queries: 2^-11 per operand (queries, centroids, weights), each rounding independent:
a score is off by about 2^-11 * sqrt(2) * S / 8, S <= 40: 3.4e-3 at most, so a mean by 7e-3 + 2^-11,
and the output's rounding adds 2^-9: 1e-2.  float16 outputs add 2^-12.
"""

import math

import numpy as np
import pytest
import torch

import tq_oracle as O
from turboquant_kv import ops
from turboquant_kv.codebook import lloyd_max_codebook, make_rotation_matrix

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = {"f32": 2e-5, "f16": 2e-5 + 2.0 ** -11, "bf16": 1e-2}


class Pools:
    """Random rows in pools, packed by the package's own stores, and their float64 values."""

    def __init__(self, seed, nblocks, H, bs, vb):
        rs = np.random.RandomState(seed)
        self.H, self.bs, self.vb, self.nb = H, bs, vb, nblocks
        n = nblocks * bs
        kc, vc = rs.randint(0, 16, (n, H, 64)), rs.randint(0, 1 << vb, (n, H, 64))
        kn = np.exp(0.3 * rs.randn(n, H)).astype(np.float32) * 6
        vn = np.exp(0.3 * rs.randn(n, H)).astype(np.float32) * 2
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(DEV)  # noqa: E731
        krows = t(O.pack_codes(kc.reshape(-1, 64).astype(np.uint8), 4)).view(n * H, 1, -1)
        vrows = t(O.pack_codes(vc.reshape(-1, 64).astype(np.uint8), vb)).view(n, H, -1)
        pairs = torch.empty(n * H, 1, 32, dtype=torch.uint8, device=DEV)
        ops.pack_decode_layout(krows, pairs, 64, 4, False, 0)
        self.kp = torch.zeros(nblocks, H, bs, 32, dtype=torch.uint8, device=DEV)
        self.kn = torch.zeros(nblocks, H, bs, device=DEV)
        self.vn = torch.zeros(nblocks, H, bs, device=DEV)
        self.vt = torch.zeros((nblocks, H, bs // 64, 512 * vb) if bs >= 64 else (nblocks, H, bs // 16, 128 * vb),
                              dtype=torch.uint8, device=DEV)
        slots = torch.arange(n, device=DEV)
        ops.paged_store(pairs.view(n, H, 32), t(kn), slots, self.kp, self.kn)
        ops.paged_store_value_tiles(vrows, t(vn), slots, self.vt, self.vn)
        self.Rk, self.Rv = make_rotation_matrix(64, seed=1).to(DEV), make_rotation_matrix(64, seed=2).to(DEV)
        self.kcen, self.vcen = lloyd_max_codebook(4, 64)[1].to(DEV), lloyd_max_codebook(vb, 64)[1].to(DEV)
        f = lambda cen, c, nn, R: (cen.double()[t(c)] @ R.double()) * t(nn).double()[..., None]  # noqa: E731
        self.k, self.v = f(self.kcen, kc, kn, self.Rk), f(self.vcen, vc, vn, self.Rv)  # [slots, H, 64]

    def args(self):
        return self.kp, self.kn, self.vt, self.vn

    def tables(self):
        return self.kcen, self.vcen, self.Rk, self.Rv


def _tables(rs, lens, bs, nblocks, width=None, fill=-1):
    perm = rs.permutation(nblocks)
    width = width or max(1, max(-(-n // bs) for n in lens))
    tab, used = np.full((len(lens), width), fill, np.int32), 0
    for i, n in enumerate(lens):
        k = -(-n // bs)
        tab[i, :k] = perm[used:used + k]
        used += k
    return tab


def want(P, q, tab, new, lens, scale, softcap=0.0, slopes=None, window=0, prefix=None, starts=None):
    """The definition in float64: outputs, log-sum-exp, and each row's largest |value row|."""
    q = q.double()
    N, Hq, _ = q.shape
    G = Hq // P.H
    out = torch.zeros(N, Hq, 64, dtype=torch.float64, device=DEV)
    lse = torch.full((N, Hq), -math.inf, dtype=torch.float64, device=DEV)
    size = torch.ones(N, Hq, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, T) in enumerate(zip(new, lens)):
        j = torch.arange(T, device=DEV)
        slot = torch.from_numpy(tab[b].astype(np.int64)).to(DEV)[j // P.bs] * P.bs + j % P.bs
        k, v = P.k[slot], P.v[slot]
        for i in range(n):
            p = T - n + i
            see = j < max(p + 1, 0 if prefix is None else prefix[b])
            if window:
                see &= j > p - window
            if starts is not None:
                see &= j >= starts[at + i]
            if not bool(see.any()):
                continue
            x = torch.einsum("hgd,thd->hgt", q[at + i].view(P.H, G, 64), k) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x + torch.as_tensor(slopes, dtype=torch.float64, device=DEV).view(P.H, G, 1) * (j - p)
            x = torch.where(see, x, -math.inf)
            lse[at + i] = torch.logsumexp(x, -1).view(Hq)
            out[at + i] = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), v).reshape(Hq, 64)
            size[at + i] = v[see].norm(dim=-1).amax(0).repeat_interleave(G)
        at += n
    return out, lse, size


def check(got, lse, ref, dt):
    out, wl, size = ref
    err = ((got.double() - out).norm(dim=-1) / size).max().item()
    assert err <= TOL[dt], err
    if lse is not None:
        seen = torch.isfinite(wl)
        assert torch.equal(seen, torch.isfinite(lse)) and bool((lse[~seen] == -math.inf).all())
        # an lse is off by what a score is (and a rounding of its own size)
        e = ((lse.double() - wl)[seen].abs() / (1 + wl[seen].abs())).max().item() if seen.any() else 0.0
        assert e <= (5e-3 if dt == "bf16" else 1e-5), e


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def run(P, rs, new, lens, Hq, dt, pad=0, groups=None, tab=None, **kw):
    tab = _tables(rs, lens, P.bs, P.nb) if tab is None else tab
    n = sum(new) + pad
    q = torch.from_numpy(rs.randn(n, Hq, 64)).to(DEV).to(DTYPES[dt])
    at = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    kw2 = dict(kw)
    for key, name in (("prefix", "prefix_lens"), ("starts", "token_starts")):
        if key in kw2:
            x = kw2.pop(key)
            kw2[name] = _ints(list(x) + [0] * (pad if key == "starts" else 0))
    if "slopes" in kw2:
        kw2["alibi_slopes"] = torch.tensor(kw2.pop("slopes"), dtype=torch.float32, device=DEV)
    args = (q, *P.args(), torch.from_numpy(tab).to(DEV), torch.from_numpy(at).to(DEV), _ints(lens))
    if groups is None:
        got, lse = ops.attention_batch_paged_dl(*args, *P.tables(), 0.125, return_lse=True, **kw2)
    else:
        got, lse = ops.attention_shared_prefix_paged_dl(*args, _ints(groups[0]), _ints(groups[1]), *P.tables(), 0.125,
                                                        return_lse=True, **kw2)
    assert got.dtype == q.dtype and got.shape == q.shape
    check(got, lse, want(P, q, tab, new, lens, 0.125, **kw), dt)
    return got, lse


@pytest.mark.parametrize("vb", [2, 3, 4])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_single_tokens(dt, bs, vb):
    """One token per sequence: contexts of none, one, around tile and block borders."""
    rs = np.random.RandomState(bs + vb)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 129, 300, 2]
    P = Pools(3, sum(-(-n // bs) for n in lens) + 3, 2, bs, vb)
    run(P, rs, [1] * len(lens), lens, 8, dt)


@pytest.mark.parametrize("H,Hq", [(1, 1), (2, 2), (2, 14), (1, 16), (1, 20), (4, 32), (3, 9)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_head_layouts(dt, H, Hq):
    rs = np.random.RandomState(Hq)
    lens = [70, 5, 200]
    P = Pools(4, 24, H, 16, 2)
    run(P, rs, [1, 1, 1], lens, Hq, dt)
    run(P, rs, [33, 5, 17], lens, Hq, dt)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lens", [([7, 1, 0, 40], [7, 300, 9, 100]), ([1], [700]), ([100], [100]),
                                      ([0, 0], [5, 0]), ([3, 3, 3], [3, 2, 500])])
def test_ragged(dt, new, lens):
    """Prompts, chunks behind a history, single and no tokens; a sequence with fewer cached
    tokens than new ones (its first rows lie before position 0 and see nothing)."""
    rs = np.random.RandomState(7)
    P = Pools(5, 64, 2, 16, 3)
    run(P, rs, new, lens, 8, dt, pad=2)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(softcap=2.0), dict(softcap=30.0), dict(window=1), dict(window=50), dict(window=10 ** 9),
    dict(slopes=[2.0 ** -i for i in range(8)]), dict(slopes=[-0.5] * 8),
    dict(prefix=[30, 0, 90, 64]), dict(prefix=[10 ** 9, -3, 100, 70]),
    dict(softcap=5.0, window=40, slopes=[0.1] * 8, prefix=[30, 5, 90, 64]),
])
def test_variants(dt, kw):
    rs = np.random.RandomState(11)
    P = Pools(6, 80, 2, 16, 2)
    run(P, rs, [20, 1, 60, 3], [50, 333, 100, 64], 8, dt, pad=1, **kw)
    kw = {k: ([v[0]] if k == "prefix" else v) for k, v in kw.items()}
    run(P, rs, [1], [777], 8, dt, **kw)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_document_starts_and_empty_rows(dt):
    """Packed documents; starts past a token's own position leave its row nothing."""
    rs = np.random.RandomState(12)
    P = Pools(7, 80, 2, 16, 4)
    new, lens = [90, 1, 1], [200, 150, 31]
    starts = [(110 + i) // 37 * 37 for i in range(90)] + [149, 31]
    starts[5], starts[50] = 10 ** 6, -4
    run(P, rs, new, lens, 8, dt, starts=starts)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vb", [2, 3, 4])
def test_long_prompts(dt, vb):
    """Enough rows for the kernel that gives each wave rows of its own."""
    rs = np.random.RandomState(13)
    P = Pools(8, 300, 8, 16 if vb != 3 else 64, vb)
    tab = _tables(rs, [1500, 10, 1100], P.bs, P.nb)
    q = torch.from_numpy(rs.randn(2600, 128, 64).astype(np.float32)).to(DEV).to(DTYPES[dt])
    at = _ints([0, 1400, 1405, 2505])
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), torch.from_numpy(tab).to(DEV), at, _ints([1500, 10, 1100]),
                                            *P.tables(), 0.125, window=700, softcap=20.0, return_lse=True)
    assert not got[2505:].any() and bool((lse[2505:] == -math.inf).all())
    # a few rows of each sequence, as single-sequence references
    for b, (a0, n, T) in enumerate([(0, 1400, 1500), (1400, 5, 10), (1405, 1100, 1100)]):
        for i in sorted({0, 1, n // 3, n - 2, n - 1}):
            ref = want(P, q[a0 + i: a0 + i + 1], tab[b:b + 1], [1], [T - n + i + 1], 0.125, softcap=20.0, window=700)
            check(got[a0 + i: a0 + i + 1], lse[a0 + i: a0 + i + 1], ref, dt)


def _shared_tables(rs, groups, shared, lens, bs, nblocks):
    tab = _tables(rs, lens, bs, nblocks)
    for g, s in enumerate(shared):
        for b in range(groups[g], groups[g + 1]):
            tab[b, :s // bs] = tab[groups[g], :s // bs]
    return tab


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("groups,shared", [([0, 6], [128]), ([0, 2, 6], [64, 192]), ([1, 4], [64]),
                                           ([0, 1, 5, 6, 6], [64, 128, 0, 64])])
def test_shared_prefix(dt, new, groups, shared):
    rs = np.random.RandomState(14)
    P = Pools(9, 200, 2, 16, 2)
    lens = [250, 230, 400, 245, 300, 232]
    tab = _shared_tables(rs, groups, shared, lens, 16, P.nb)
    run(P, rs, [new] * 6, lens, 8, dt, pad=2, groups=(groups, shared), tab=tab)


@pytest.mark.parametrize("kw", [dict(window=100), dict(softcap=3.0, slopes=[0.05] * 8), dict(prefix=[150] * 4),
                                dict(prefix=[20, 260, 1, 64], window=130)])
def test_shared_prefix_variants(kw):
    """Windows that leave the prefix out, prefixes that end inside it, contexts inside it."""
    rs = np.random.RandomState(15)
    P = Pools(10, 120, 2, 32, 3)
    lens = [260, 130, 100, 500]
    tab = _shared_tables(rs, [0, 4], [128], lens, 32, P.nb)
    run(P, rs, [2, 1, 1, 9], lens, 8, "f32", groups=([0, 4], [128]), tab=tab, **kw)
    starts = [0, 129, 5, 100, 3, 499, 10 ** 6] + [200] * 6
    run(P, rs, [2, 1, 1, 9], lens, 8, "f32", groups=([0, 4], [128]), tab=tab, starts=starts)


def test_long_context_cut_between_workgroups():
    """One long sequence among short ones: its tiles are cut between many workgroups."""
    rs = np.random.RandomState(16)
    P = Pools(11, 1100, 1, 16, 2)
    for dt in ("f32", "bf16"):
        run(P, rs, [1, 1, 1], [16000, 5, 800], 4, dt, softcap=30.0)
        run(P, rs, [30, 1, 2], [16000, 5, 800], 4, dt)


def test_strided_queries_and_outputs_and_padding():
    """Queries sliced out of a fused projection; a given output keeps its rows behind the last
    sequence; an lse of -inf there."""
    rs = np.random.RandomState(17)
    P = Pools(12, 40, 2, 16, 2)
    lens, new = [100, 60], [2, 1]
    tab = _tables(rs, lens, 16, P.nb)
    qkv = torch.from_numpy(rs.randn(5, 12, 64).astype(np.float32)).to(DEV).bfloat16()
    q = qkv[:, :8]
    dst = torch.full((5, 10, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    out = dst[:, :8]
    a = (torch.from_numpy(tab).to(DEV), _ints([0, 2, 3]), _ints(lens), *P.tables(), 0.125)
    r, lse = ops.attention_batch_paged_dl(q, *P.args(), *a, out=out, return_lse=True)
    assert r is out
    check(out[:3], lse[:3], want(P, q[:3], tab, new, lens, 0.125), "bf16")
    assert bool((dst[3:] == 7).all()) and bool((dst[:, 8:] == 7).all()) and bool((lse[3:] == -math.inf).all())
    again = ops.attention_batch_paged_dl(q.contiguous(), *P.args(), *a)
    assert torch.equal(again[:3], out[:3]) and not again[3:].any()
    odd = torch.zeros(5 * 12 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(5, 12, 64)  # 2-byte aligned
    odd.copy_(qkv)
    assert torch.equal(ops.attention_batch_paged_dl(odd[:, :8], *P.args(), *a), again)


def test_stale_rows_hold_nan():
    """NaN and inf norms in masked places: past the context, behind a window, and a later token
    that earlier rows of its tile do not see."""
    rs = np.random.RandomState(18)
    P = Pools(13, 30, 2, 16, 2)
    lens, new = [70, 33], [4, 1]
    tab = _tables(rs, lens, 16, P.nb)
    for b, T in enumerate(lens):
        blk, at = int(tab[b, (T - 1) // 16]), T % 16
        if at:
            P.kn[blk, :, at:] = math.nan
            P.vn[blk, :, at:] = math.inf
    run(P, rs, new, lens, 8, "f32", tab=tab)
    run(P, rs, new, lens, 8, "bf16", tab=tab)
    P.kn[int(tab[0, 0]), :, :8] = math.nan
    P.vn[int(tab[0, 0]), :, :8] = math.nan
    run(P, rs, new, lens, 8, "f32", tab=tab, window=50)
    # the last new token's norms: rows before it must not see them
    blk = int(tab[0, 69 // 16])
    P.kn[blk, :, 69 % 16] = math.nan
    P.vn[blk, :, 69 % 16] = math.inf
    q = torch.from_numpy(rs.randn(5, 8, 64)).to(DEV).float()
    got = ops.attention_batch_paged_dl(q, *P.args(), torch.from_numpy(tab).to(DEV), _ints([0, 4, 5]), _ints(lens),
                                       *P.tables(), 0.125, window=50)
    ref = want(P, q[:3], tab[:1], [3], [69], 0.125, window=50)
    check(got[:3], None, ref, "f32")
    assert bool(torch.isnan(got[3]).all())


def test_corrupt_tables_and_lengths_stay_inside():
    """Block ids, lengths and starts out of range are clamped: nothing outside is read and
    untouched sequences keep their results."""
    rs = np.random.RandomState(19)
    P = Pools(14, 30, 2, 16, 2)
    lens, new = [70, 33], [2, 1]
    tab = _tables(rs, lens, 16, P.nb)
    q = torch.from_numpy(rs.randn(3, 8, 64)).to(DEV).float()
    bad = tab.copy()
    bad[0, 1], bad[0, 2] = 10 ** 9, -7
    t = lambda x: torch.from_numpy(x).to(DEV)  # noqa: E731
    got = ops.attention_batch_paged_dl(q, *P.args(), t(bad), _ints([0, 2, 3]), _ints([10 ** 9, 33]), *P.tables(), 0.125)
    check(got[2:], None, tuple(x[2:] for x in want(P, q, tab, new, lens, 0.125)), "f32")
    for starts in ([0, 99, -5], [3, 2, 1], [-4, 1, 70000], [5, 5, 5]):
        for extra in ((), (_ints([0, 2]), _ints([16])), (_ints([2, -1, 9]), _ints([10 ** 9, -3]))):
            fn = ops.attention_shared_prefix_paged_dl if extra else ops.attention_batch_paged_dl
            fn(q, *P.args(), t(tab), _ints(starts), _ints([-5, 33]), *extra, *P.tables(), 0.125)
    torch.cuda.synchronize()


def test_no_sequences_no_tokens_no_blocks():
    P = Pools(15, 4, 2, 16, 2)
    q = torch.randn(3, 8, 64, device=DEV)
    none = torch.empty(0, 5, dtype=torch.int32, device=DEV)
    got, lse = ops.attention_batch_paged_dl(q, *P.args(), none, _ints([0]), _ints([]), *P.tables(), 0.125, return_lse=True)
    assert not got.any() and bool((lse == -math.inf).all())
    got = ops.attention_batch_paged_dl(q[:0], *P.args(), none, _ints([0]), _ints([]), *P.tables(), 0.125)
    assert got.shape == (0, 8, 64)
    empty = torch.empty(1, 0, dtype=torch.int32, device=DEV)
    got = ops.attention_batch_paged_dl(q, *P.args(), empty, _ints([0, 2]), _ints([9]), *P.tables(), 0.125)
    assert not got.any()


@pytest.mark.parametrize("shared", [False, True])
def test_captured_and_replayed(shared):
    """A captured call replays with the lengths and queries its tensors hold then."""
    rs = np.random.RandomState(20)
    P = Pools(16, 120, 2, 16, 2)
    lens = [300, 280, 290]
    tab = _shared_tables(rs, [0, 3], [128], lens, 16, P.nb)
    q = torch.from_numpy(rs.randn(4, 8, 64)).to(DEV).bfloat16()
    t, at, sl = torch.from_numpy(tab).to(DEV), _ints([0, 1, 2, 3]), _ints(lens)
    extra = (_ints([0, 3]), _ints([128])) if shared else ()
    fn = ops.attention_shared_prefix_paged_dl if shared else ops.attention_batch_paged_dl
    call = lambda: fn(q, *P.args(), t, at, sl, *extra, *P.tables(), 0.125, softcap=20.0)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        sl.copy_(_ints([290 + step, 200 + 20 * step, 140 + step]))
        q.copy_(torch.from_numpy(rs.randn(4, 8, 64)))
        graph.replay()
        got = out.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_streams_side_by_side():
    """Two calls at once on streams of their own, each with its own workspace."""
    rs = np.random.RandomState(21)
    P = Pools(17, 200, 2, 16, 2)
    lens = [1500, 900]
    t = torch.from_numpy(_tables(rs, lens, 16, P.nb)).to(DEV)
    q = [torch.from_numpy(rs.randn(2, 8, 64)).to(DEV).float() for _ in range(2)]
    at, sl = _ints([0, 1, 2]), _ints(lens)
    call = lambda x: ops.attention_batch_paged_dl(x, *P.args(), t, at, sl, *P.tables(), 0.125)  # noqa: E731
    ref = [call(x) for x in q]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in q], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(q[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, ref[i]) for x in got[i])


def test_refusals():
    P = Pools(18, 4, 2, 16, 2)
    q = torch.randn(2, 8, 64, device=DEV)
    tab, at, sl = torch.zeros(1, 2, dtype=torch.int32, device=DEV), _ints([0, 2]), _ints([20])
    ok = dict(q=q, tab=tab, at=at, sl=sl)

    def call(P=P, kw=None, **c):
        c = {**ok, **c}
        return ops.attention_batch_paged_dl(c["q"], *P.args(), c["tab"], c["at"], c["sl"], *P.tables(), 0.125, **(kw or {}))
    call()
    for c in (dict(q=q.cpu()), dict(q=q.double()), dict(q=q[0]), dict(q=q[:, :7]), dict(q=q[:, :, :32]),
              dict(tab=tab[0]), dict(tab=tab.float()), dict(at=at[:1]), dict(sl=_ints([1, 2])),
              dict(kw=dict(softcap=-1.0)), dict(kw=dict(softcap=math.inf)), dict(kw=dict(window=-1)),
              dict(kw=dict(alibi_slopes=torch.ones(7, device=DEV))), dict(kw=dict(prefix_lens=_ints([1, 2]))),
              dict(kw=dict(token_starts=_ints([1]))), dict(kw=dict(out=torch.empty(2, 8, 64, device=DEV).half())),
              dict(kw=dict(out=torch.empty(3, 8, 64, device=DEV)))):
        with pytest.raises(RuntimeError):
            call(**c)
    for gs, sh in ((_ints([0, 1]), _ints([1, 2])), (_ints([0]), _ints([4]))):
        with pytest.raises(RuntimeError):
            ops.attention_shared_prefix_paged_dl(q, *P.args(), tab, at, sl, gs, sh, *P.tables(), 0.125)
