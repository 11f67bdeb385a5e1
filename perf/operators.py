"""The operators of a paged serving step over packed KV caches that this package is timed on.

A case is a dict of plain values; `kind` names the operator:

  plan    a step's block tables and slot map from the requests' lengths: which block each
          new token's request takes from the free list, and where each token is stored
  groups  the runs of neighbouring requests whose block tables begin with the same blocks
  attn    attention of a ragged batch (prompts, chunks and single tokens together) over the
          packed pools, its scores capped by a tanh, biased by distance (ALiBi), and masked
          by a window, a bidirectional prefix or per-token document starts
  shared  the same attention for batches whose requests share a long prefix, which is read
          once per group of requests

A packed pool holds 4-bit key codes as pair bytes [blocks, H, block, 32], 2- to 4-bit value
codes as tiles of 64 tokens (blocks of 64) or sub-blocks of 16 tokens (blocks of 16 and 32),
and a norm per token and head; a row is norm * centroid[code] rotated by an orthogonal R.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
D = 64  # head size of the packed pools
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}
I32, I64, F32 = torch.int32, torch.int64, torch.float32


def _plan(name, **kw):
    c = dict(name=name, kind="plan", requests=16, context=4096, new=1, prompts=0, block=16, pad=0, mix=1)
    c.update(kw)
    return c


def _groups(name, **kw):
    c = dict(name=name, kind="groups", requests=32, context=4096, groups=4, shared=2048, block=16,
             least=256, mix=1)
    c.update(kw)
    return c


def _attn(name, kind="attn", **kw):
    # `prompts` sequences of up to `new` new tokens, the others with one (decode) each
    c = dict(name=name, kind=kind, batch=1, prompts=0, new=1, context=1000, hq=32, hkv=8, vbits=2,
             block=16, dtype="bfloat16", softcap=0.0, alibi=False, window=0, prefix=False, docs=0,
             pad=0, lse=False, mix=1)
    c.update(kw)
    return c


def _shared(name, **kw):
    c = dict(batch=16, context=2560, groups=1, shared=2048)
    c.update(kw)
    return _attn(name, "shared", **c)


def listed():
    return [
        # a small serving batch's decode step: every request takes one slot, few take a block
        _plan("plan_decode_16"),
        # a large engine's step: a thousand requests, some of them prompt chunks, padded to a
        # graph's token count
        _plan("plan_mixed_1024", requests=1024, context=8192, new=512, prompts=64, pad=777),
        # a batch of requests behind a few system prompts
        _groups("groups_32_4k"),
        # a large engine's tables at long context, one system prompt for most requests
        _groups("groups_1024_16k", requests=1024, context=16_384, groups=2, shared=8192),
        # one request's decode step at a short context, capped scores: the latency of a layer
        _attn("attn_decode_b1_1k", softcap=50.0),
        # a serving batch's decode step, capped scores, a graph's padding rows behind it
        _attn("attn_decode_b48_8k", batch=48, context=8192, softcap=50.0, vbits=3, pad=3),
        # long contexts with a distance bias, 16-bit floats, blocks of 64 tokens
        _attn("attn_decode_b32_32k_alibi", batch=32, context=32_768, dtype="float16", alibi=True,
              vbits=4, block=64),
        # ragged prompts of a model with sliding windows and capped scores
        _attn("attn_prefill_b4_4k", batch=4, prompts=4, new=4096, context=4096, window=1024,
              softcap=30.0),
        # a mixed step in float32: two prompt chunks with a bidirectional prefix and packed
        # documents behind long histories, and decode tokens of six other requests
        _attn("attn_mixed_b8_12k", batch=8, prompts=2, new=512, context=12_288, dtype="float32",
              prefix=True, docs=3000, block=32, lse=True),
        # a few requests behind one prompt
        _shared("shared_b16_2k"),
        # a large batch behind a long document, 3-bit values
        _shared("shared_b128_16k", batch=128, context=17_408, shared=16_384, vbits=3),
        # four prompts, four new tokens per request (speculative decoding), float16
        _shared("shared_g4_b64_8k", batch=64, prompts=64, new=4, context=10_240, groups=4,
                shared=8192, dtype="float16", lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["plan", "groups", "attn", "attn", "attn", "shared", "shared"])
    mix = rng.randrange(1, 1 << 20)
    block = rng.choice([16, 16, 32, 64])
    if kind == "plan":
        n = _log(rng, 1, 1024)
        prompts = 0 if rng.random() < 0.4 else rng.randint(1, max(1, n // 16))
        return _plan(None, requests=n, context=_log(rng, 700, 8192), new=_log(rng, 2, 512) if prompts else 1,
                     prompts=prompts, block=block, pad=rng.choice([0, 0, rng.randint(1, 300)]), mix=mix)
    if kind == "groups":
        n = _log(rng, 2, 1024)
        context = _log(rng, 2000, 16_384)
        return _groups(None, requests=n, context=context, groups=rng.randint(1, max(1, min(8, n // 2))),
                       shared=rng.randint(context // 2, context) // block * block, block=block,
                       least=rng.choice([1, 64, 256]), mix=mix)
    hq, hkv = rng.choice([(32, 8), (32, 8), (8, 8), (28, 4), (16, 2), (20, 1), (6, 2)])
    c = dict(hq=hq, hkv=hkv, vbits=rng.choice([2, 3, 4]), block=block, mix=mix,
             dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
             pad=rng.choice([0, 0, rng.randint(1, 9)]))
    c["softcap"] = rng.choice([0.0, 30.0, 50.0])
    c["alibi"] = rng.random() < 0.25
    c["window"] = rng.choice([0, 0, 0, rng.randint(1, 3000)])
    c["prefix"] = rng.random() < 0.2
    c["docs"] = rng.choice([0, 0, 0, rng.randint(40, 4000)])
    c["lse"] = c["dtype"] != "bfloat16" and rng.random() < 0.5
    if kind == "shared":
        c["window"] = c["docs"] = 0
        c["new"] = rng.choice([1, 1, 1, 2, 4])
        c["batch"] = _log(rng, 2, 128 // c["new"])
        c["groups"] = rng.randint(1, max(1, min(4, c["batch"] // 2)))
        c["shared"] = max(1, _log(rng, 64, 16_384) // block) * block
        c["prompts"] = c["batch"] if c["new"] > 1 else 0
        c["context"] = c["shared"] + c["new"] + _log(rng, 1, 1024)
        return _attn(None, "shared", **c)
    if rng.random() < 0.5:  # single tokens
        c["batch"] = _log(rng, 1, 64)
        c["context"] = max(2, min(_log(rng, 2, 32_768), (1 << 20) // c["batch"]))
    else:
        c["batch"] = rng.choice([1, 2, 4, 8])
        c["prompts"] = rng.randint(1, c["batch"])
        c["new"] = _log(rng, 2, 4096 // c["batch"])
        c["context"] = c["new"] + (0 if rng.random() < 0.5 else _log(rng, 1, 8192 // c["batch"]))
    return _attn(None, **c)


# ------------------------------------------------------------------------- a case's lengths

def _rng(case):
    return random.Random(case["mix"] * 1_000_003 + case["context"])


def _plan_lengths(case):
    """Per request: new tokens, and tokens that its cache holds before them."""
    r, n = _rng(case), case["requests"]
    new = [r.randint(1, case["new"]) if i < case["prompts"] else 1 for i in range(n)]
    r.shuffle(new)
    old = [r.randint(0, max(0, case["context"] - k)) for k in new]
    return new, old


def _group_members(case, n):
    """The first request of each group, and n: groups of about the same size."""
    return [n * g // case["groups"] for g in range(case["groups"] + 1)]


def _table_groups(case, seed):
    """Of a `groups` case: the first request of each group, the tokens it shares (whole
    blocks), and the requests' context lengths."""
    r, n, bs = random.Random(seed * 7919 + case["mix"]), case["requests"], case["block"]
    at = _group_members(case, n)
    at[1:-1] = [r.randint((a + b + 1) // 2, b) for a, b in zip(at[:-2], at[1:-1])]
    most = case["shared"] // bs
    shared = [r.randint((most + 1) // 2, most) * bs for _ in at[1:]]
    return at, shared, [r.randint(case["context"] // 2, case["context"]) for _ in range(n)]


def _group_shared(case):
    """Tokens each group shares, whole blocks: the first group's is the longest."""
    r, bs = _rng(case), case["block"]
    most = case["shared"] // bs
    return [most * bs] + [r.randint(most // 2, most) * bs for _ in range(case["groups"] - 1)]


def _attn_lengths(case):
    """Per sequence: new tokens, and tokens of its context (the new ones included)."""
    r, n = _rng(case), case["batch"]
    new = [case["new"] if i == 0 else r.randint(max(1, case["new"] // 2), case["new"])
           for i in range(case["prompts"])]
    new += [1] * (n - case["prompts"])
    least = [k for k in new]
    if case["kind"] == "shared":
        at, sh = _group_members(case, n), _group_shared(case)
        least = [sh[max(g for g in range(case["groups"]) if at[g] <= i)] + new[i] for i in range(n)]
    lens = [case["context"] if i == 0 else
            r.randint(min(case["context"], max(least[i], case["context"] // 4)), case["context"])
            for i in range(n)]
    return new, lens


def _prefix_lens(case, new, lens):
    """The part of each context that all its tokens see: the history and half of the new."""
    return [t - k + k // 2 for k, t in zip(new, lens)] if case["prefix"] else None


def _slopes(hq):
    return [2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)]


# ----------------------------------------------------------------------------------- inputs

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000 + salt)


def _ints(values, dtype=I32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _codebook(bits):
    """Boundaries and centroids of a Lloyd-Max quantizer of N(0, 1 / D), in 64 bits."""
    n = 1 << bits
    c = torch.linspace(-2.0, 2.0, n, dtype=torch.float64)
    phi = lambda x: torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)  # noqa: E731
    cdf = lambda x: 0.5 * torch.erfc(-x / math.sqrt(2))  # noqa: E731
    inf = torch.tensor([math.inf], dtype=torch.float64)
    for _ in range(300):
        b = torch.cat([-inf, (c[1:] + c[:-1]) / 2, inf])
        c = (phi(b[:-1]) - phi(b[1:])) / (cdf(b[1:]) - cdf(b[:-1]))
    return ((c[1:] + c[:-1]) / 2).to(DEV, F32), (c / math.sqrt(D)).to(DEV, F32)


def _codes(bits, shape, seed, salt):
    """Codes of rotated unit vectors: their coordinates are near N(0, 1 / D)."""
    bounds, g = _codebook(bits)[0], _gen(seed, salt)
    out = torch.empty(shape, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, shape[0], step):
        x = torch.randn((min(step, shape[0] - at),) + shape[1:], generator=g, device=DEV)
        out[at: at + step] = torch.bucketize(x, bounds).to(torch.uint8)
    return out


def _rotation(seed, salt):
    q, r = torch.linalg.qr(torch.randn(D, D, generator=_gen(seed, salt), device=DEV, dtype=torch.float64).cpu())
    return (q * torch.sign(torch.diagonal(r))).to(DEV, F32)


def _pack_keys(codes):
    return codes[..., 0::2] << 4 | codes[..., 1::2]


def _pack_values(codes, bits):
    """[blocks, H, block, D] codes as the pools hold them: token 16 m + 4 s + t, dim 16 g + c."""
    nb, h, bs, _ = codes.shape
    if bits == 2:  # a byte holds the codes of four tokens
        x = codes.view(nb, h, bs // 16, 4, 4, 4, 16)                    # m s t g c
        x = x[..., 0, :, :] | x[..., 1, :, :] << 2 | x[..., 2, :, :] << 4 | x[..., 3, :, :] << 6
        x = x.unsqueeze(4)                                              # m s 1 g c
    else:  # a byte holds a pair of tokens' codes
        x = codes.view(nb, h, bs // 16, 4, 2, 2, 4, 16)                 # m s j pair g c
        x = x[..., 0, :, :] | x[..., 1, :, :] << bits                   # m s j g c
    if bits == 3:  # six bits a byte: dims 48.. take the top bits of the three others
        y = x[..., 3, :]
        x = torch.stack([x[..., i, :] | (y >> (2 * i) & 3) << 6 for i in range(3)], -2)
    if bs >= 64:  # a tile: lane (s, c)'s 32-bit words, the first four of each lane before the rest
        x = x.view(nb, h, bs // 64, 4, *x.shape[3:])                    # tile m s j g c
        if bits == 2:
            return x.permute(0, 1, 2, 4, 7, 3, 5, 6).reshape(nb, h, bs // 64, 1024).contiguous()
        x = x.view(nb, h, bs // 64, 2, 2, *x.shape[4:])                 # tile M m2 s j g c
        x = x.permute(0, 1, 2, 5, 8, 3, 7, 4, 6)                        # tile s c M g m2 j
        x = x.reshape(nb, h, bs // 64, 64, -1)
        return torch.cat([x[..., :16].flatten(3), x[..., 16:].flatten(3)], 3).contiguous()
    x = x.permute(0, 1, 2, 3, 6, 5, 4).reshape(nb, h, bs // 16, 64, -1)  # m (s c) (g j)
    if bits == 3:
        return torch.cat([x[..., :4].flatten(3), x[..., 4:].flatten(3)], 3).contiguous()
    return x.flatten(3).contiguous()


def _tables(case, seed, lens):
    """Shuffled block tables of the sequences (shared blocks first within a group), and the
    number of blocks in the pool."""
    bs, n = case["block"], len(lens)
    need = [-(-t // bs) for t in lens]
    at, sh = [], []
    if case["kind"] == "shared":
        at, sh = _group_members(case, n), _group_shared(case)
    if case["kind"] == "groups":
        at, sh, _ = _table_groups(case, seed)
    sh = [s // bs for s in sh]
    rows, used = [], 0
    for i in range(n):
        g = max([g for g in range(len(sh)) if at[g] <= i], default=-1)
        common = []
        if g >= 0:
            if i == at[g]:
                first = list(range(used, used + sh[g]))
                used += sh[g]
            common = first[: need[i]]
        rows.append(common + list(range(used, used + need[i] - len(common))))
        used += need[i] - len(common)
    width = max(need) + 3
    total = used + 5
    order = torch.randperm(total, generator=_gen(seed, 6), device=DEV)
    tab = torch.zeros(n, width, dtype=I64)
    for i, row in enumerate(rows):
        tab[i, : len(row)] = torch.tensor(row, dtype=I64)
    return order[tab.to(DEV)].to(I32), total


def _starts(counts):
    at = [0]
    for k in counts:
        at.append(at[-1] + k)
    return at


def _make(case, seed):
    """An attention case's inputs, and the pools' codes before they are packed."""
    new, lens = _attn_lengths(case)
    tables, blocks = _tables(case, seed, lens)
    h, bs, dt = case["hkv"], case["block"], DTYPES[case["dtype"]]
    shape = (blocks, h, bs, D)
    kc, vc = _codes(4, shape, seed, 1), _codes(case["vbits"], shape, seed, 2)
    norm = lambda mean, salt: mean * torch.exp(  # noqa: E731
        0.25 * torch.randn(shape[:3], generator=_gen(seed, salt), device=DEV))
    at = _starts(new)
    q = torch.randn(at[-1] + case["pad"], case["hq"], D, generator=_gen(seed, 5), device=DEV)
    pre = _prefix_lens(case, new, lens)
    st = dict(
        case=case, q=(1.25 * q).to(dt), kp=_pack_keys(kc), kn=norm(8.0, 3), vt=_pack_values(vc, case["vbits"]),
        vn=norm(4.0, 4), tables=tables, qsl=_ints(at), lens=_ints(lens), kcen=_codebook(4)[1],
        vcen=_codebook(case["vbits"])[1], rk=_rotation(seed, 7), rv=_rotation(seed, 8),
        slopes=torch.tensor(_slopes(case["hq"]), dtype=F32, device=DEV) if case["alibi"] else None,
        prefix=None if pre is None else _ints(pre), starts=None, most=max(new))
    if case["docs"]:  # the first token of each new token's document
        pos = [t - k + i for k, t in zip(new, lens) for i in range(k)]
        st["starts"] = _ints([p // case["docs"] * case["docs"] for p in pos] + [0] * case["pad"])
    if case["kind"] == "shared":
        st["groups"] = _ints(_group_members(case, case["batch"]))
        st["shared"] = _ints(_group_shared(case))
    return st, kc, vc


def prepare(case, seed):
    if case["kind"] == "plan":
        new, old = _plan_lengths(case)
        bs = case["block"]
        tables, blocks = _tables(case, seed, [max(1, a + b) for a, b in zip(old, new)])
        held = torch.arange(tables.shape[1], device=DEV) < _ints([-(-t // bs) for t in old])[:, None]
        free = torch.ones(blocks, dtype=torch.bool, device=DEV)
        free[tables[held].long()] = False
        free = free.nonzero().view(-1)
        free = free[torch.randperm(free.numel(), generator=_gen(seed, 7), device=DEV)].to(I32)
        return dict(case=case, new=_ints(new), old=_ints(old), tables=torch.where(held, tables, -1), free=free,
                    tokens=sum(new) + case["pad"])
    if case["kind"] == "groups":
        lens = _table_groups(case, seed)[2]
        tables, _ = _tables(case, seed, lens)
        return dict(case=case, tables=tables, lens=_ints(lens))
    return _make(case, seed)[0]


# -------------------------------------------------------------------------- the plain forms

def _plan_plain(s):
    bs, n, dev = s["case"]["block"], s["tokens"], DEV
    new, old, tables, free = s["new"].long(), s["old"].long(), s["tables"], s["free"].long()
    width = tables.shape[1]
    at = torch.cat([new.new_zeros(1), new.cumsum(0)])
    total = old + new
    held, need = (old + bs - 1) // bs, (total + bs - 1) // bs
    takes = need - held
    first = takes.cumsum(0) - takes  # of the free list, per request
    j = torch.arange(width, device=dev)
    fresh = (j >= held[:, None]) & (j < need[:, None])
    tables.copy_(torch.where(fresh, free[(first[:, None] + j - held[:, None]).clamp(0, free.numel() - 1)], tables.long()))
    i = torch.arange(n, device=dev)
    req = torch.searchsorted(at[1:].contiguous(), i, right=True)
    real = i < at[-1]
    req = req.clamp(max=new.numel() - 1)
    pos = old[req] + i - at[req]
    slot = tables.long()[req, (pos // bs).clamp(0, width - 1)] * bs + pos % bs
    return dict(query_start_loc=at.to(I32), seq_lens=total.to(I32), slot_mapping=torch.where(real, slot, -1),
                positions=torch.where(real, pos, 0), token_request=torch.where(real, req, -1).to(I32),
                blocks_used=takes.sum().to(I32).reshape(1), block_tables=tables)


def _groups_plain(s):
    bs, least, tables, lens = s["case"]["block"], s["case"]["least"], s["tables"], s["lens"]
    n, width = tables.shape
    full = torch.minimum(lens[1:], lens[:-1]) // bs
    same = (tables[1:] == tables[:-1]) & (torch.arange(width, device=DEV) < full[:, None])
    common = same.to(I32).cumprod(1).sum(1) * bs
    joined = common >= least
    group = torch.cat([joined.new_zeros(1).long(), (~joined).long().cumsum(0)])
    opens = torch.cat([joined.new_ones(1), ~joined])
    starts = torch.full((n + 1,), n, dtype=I64, device=DEV)
    at = torch.arange(n, device=DEV)
    starts.scatter_reduce_(0, group, torch.where(opens, at, n), "amin")
    far = torch.full((n,), 1 << 40, dtype=I64, device=DEV)
    far.scatter_reduce_(0, group[1:], torch.where(joined, common, 1 << 40), "amin")
    return dict(group_start_loc=starts.to(I32), shared_lens=torch.where(far < 1 << 40, far, 0).to(I32))


def _unpack_values(tiles, bits, bs):
    """[..., block / 64 or block / 16, width] bytes -> [..., block, D] codes."""
    t, d = torch.arange(bs, device=DEV)[:, None], torch.arange(D, device=DEV)[None, :]
    m, s, t4 = t // 16, t // 4 % 4, t % 4
    g, lane = d // 16, 16 * s + d % 16
    flat, wide, m4, m2, j = tiles.flatten(-2), tiles.shape[-1], m % 4, m % 2, t4 // 2
    base = (t // 64 if bs >= 64 else m) * wide
    if bits == 2:
        at = 16 * lane + 4 * m4 + g if bs >= 64 else 4 * lane + g
        return flat[..., base + at] >> (2 * t4).to(torch.uint8) & 3
    per = 4 if bits == 4 else 3  # words of a lane for 32 tokens
    word = lambda i: ((m4 // 2) * per + i)  # noqa: E731
    if bs >= 64:
        at = lambda i: torch.where(word(i) < 4, 16 * lane + 4 * word(i),  # noqa: E731
                                   1024 + (8 * bits - 16) * lane + 4 * (word(i) - 4)) + 2 * m2 + j
    elif bits == 4:
        at = lambda i: 8 * lane + 2 * i + j  # noqa: E731
    else:
        at = lambda i: torch.where(i < 2, 4 * lane + 2 * i, 256 + 2 * lane) + j  # noqa: E731
    half = (bits * (t4 % 2)).to(torch.uint8)
    if bits == 4:
        return flat[..., base + at(g)] >> half & 15
    low = flat[..., base + at(g.clamp(max=2))] & 63
    zero = torch.zeros_like(g)
    top = (flat[..., base + at(zero)] >> 6 | flat[..., base + at(zero + 1)] >> 6 << 2
           | flat[..., base + at(zero + 2)] >> 6 << 4)
    return torch.where(g < 3, low, top) >> half & 7


def _attn_plain(s):
    """Every sequence padded to the longest: rows dequantized (in the rotated space, where the
    query is taken too), scores, masks, softmax and values in float32."""
    c, q, tables = s["case"], s["q"].float(), s["tables"].long()
    hq, h, bs, most = c["hq"], c["hkv"], c["block"], s["most"]
    b, g, scale = tables.shape[0], hq // h, 1.0 / math.sqrt(D)
    span = tables.shape[1] * bs
    row = lambda x: x[tables].transpose(1, 2).reshape(b, h, span, -1)  # noqa: E731
    pairs = row(s["kp"]).long()
    keys = s["kcen"][torch.stack([pairs >> 4, pairs & 15], -1).flatten(-2)] * row(s["kn"].unsqueeze(-1))
    del pairs
    at, lens = s["qsl"].long(), s["lens"].long()
    count = at[1:] - at[:-1]
    i = torch.arange(most, device=DEV)
    live = i < count[:, None]                                            # [b, most]
    token = torch.where(live, at[:-1, None] + i, 0)
    qr = (q @ s["rk"].t())[token].view(b, most, h, g, D).permute(0, 2, 3, 1, 4).reshape(b, h, g * most, D)
    x = (qr @ keys.transpose(2, 3)).view(b, h, g, most, span) * scale
    del keys
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    qpos, kpos = (lens - count)[:, None] + i, torch.arange(span, device=DEV)
    if s["slopes"] is not None:
        x = x + s["slopes"].view(h, g, 1, 1) * (kpos - qpos[..., None]).float()[:, None, None]
    hi = qpos + 1
    if s["prefix"] is not None:
        hi = torch.maximum(hi, s["prefix"].long()[:, None])
    hi = torch.minimum(hi, lens[:, None])
    lo = qpos - c["window"] + 1 if c["window"] else torch.zeros_like(qpos)
    if s["starts"] is not None:
        lo = torch.maximum(lo, s["starts"].long()[token])
    seen = ((kpos >= lo[..., None]) & (kpos < hi[..., None]) & live[..., None])[:, None, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    del x, seen
    total = w.sum(-1, keepdim=True)
    vals = s["vcen"][row(_unpack_values(s["vt"], c["vbits"], bs)).long()] * row(s["vn"].unsqueeze(-1))
    o = (w.view(b, h, g * most, span) @ vals).view(b, h, g, most, D) / torch.where(total > 0, total, 1.0)
    o = (o @ s["rv"]).permute(0, 3, 1, 2, 4).reshape(b * most, hq, D)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(b * most, hq)
    n = q.shape[0]
    dst = torch.where(live, token, n).reshape(-1)
    out = q.new_zeros(n + 1, hq, D).index_copy_(0, dst, o)[:n].to(s["q"].dtype)
    if not c["lse"]:
        return [out]
    return [out, q.new_full((n + 1, hq), -math.inf).index_copy_(0, dst, lse)[:n]]


# ---------------------------------------------------------------------- the package's calls

def _package():
    path = os.path.join(os.getcwd(), "turboquant-kv_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from turboquant_kv import ops
    return ops


def _run_own(s):
    ops, c = _package(), s["case"]
    if c["kind"] == "plan":
        p = ops.paged_batch_plan(s["new"], s["old"], s["tables"], s["free"], c["block"], s["tokens"])
        return dict(query_start_loc=p[0], seq_lens=p[1], slot_mapping=p[2], positions=p[3],
                    token_request=p[4], blocks_used=p[5], block_tables=s["tables"])
    if c["kind"] == "groups":
        p = ops.shared_prefix_groups(s["tables"], s["lens"], c["block"], c["least"])
        return dict(group_start_loc=p[0], shared_lens=p[1])
    args = [s["q"], s["kp"], s["kn"], s["vt"], s["vn"], s["tables"], s["qsl"], s["lens"]]
    fixed = [s["kcen"], s["vcen"], s["rk"], s["rv"], 1.0 / math.sqrt(D)]
    kw = dict(softcap=c["softcap"], alibi_slopes=s["slopes"], window=c["window"], prefix_lens=s["prefix"],
              token_starts=s["starts"], return_lse=c["lse"])
    if c["kind"] == "shared":
        out = ops.attention_shared_prefix_paged_dl(*args, s["groups"], s["shared"], *fixed, **kw)
    else:
        out = ops.attention_batch_paged_dl(*args, *fixed, **kw)
    return list(out) if c["lse"] else [out]


def run(state):
    with torch.no_grad():
        if own:
            return _run_own(state)
        return {"plan": _plan_plain, "groups": _groups_plain}.get(state["case"]["kind"], _attn_plain)(state)


# ------------------------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "plan":
        new, old = _plan_lengths(case)
        bs, n = case["block"], case["requests"]
        fresh = sum(-(-(a + b) // bs) - -(-a // bs) for a, b in zip(old, new))
        tokens = sum(new) + case["pad"]
        # lengths in; a block id in and out for each fresh block; the part of the tables that the
        # new tokens' slots name; per token a slot, a position and a request out
        return {"bytes": 4 * (4 * n + 2 * fresh + n) + 20 * tokens, "flops": 0}
    if case["kind"] == "groups":
        # the tables up to where neighbours differ: three quarters of `shared` on average
        n = case["requests"]
        blocks = n * (3 * case["shared"] // (4 * case["block"]) + 1)
        return {"bytes": 4 * (blocks + 4 * n), "flops": 0}
    new, lens = _attn_lengths(case)
    hq, h, sz = case["hq"], case["hkv"], SIZES[case["dtype"]]
    pre = _prefix_lens(case, new, lens)
    at, sh = [0, case["batch"]], [0]
    if case["kind"] == "shared":
        at, sh = _group_members(case, case["batch"]), _group_shared(case)
    rows = pairs = 0
    for g in range(len(sh)):
        rows += sh[g]  # read once for its group
        for b in range(at[g], at[g + 1]):
            first = lens[b]
            for i in range(new[b]):
                pos = lens[b] - new[b] + i
                hi = max(pos + 1, pre[b]) if pre else pos + 1
                lo = max(0, pos - case["window"] + 1) if case["window"] else 0
                lo = max(lo, pos // case["docs"] * case["docs"]) if case["docs"] else lo
                pairs += hi - lo
                first = min(first, lo)
            rows += lens[b] - max(first, sh[g])
    tokens = sum(new) + case["pad"]
    return {"bytes": rows * h * (32 + 8 * case["vbits"] + 8) + 2 * tokens * hq * D * sz,
            "flops": 4 * D * hq * pairs + 4 * D * D * hq * sum(new)}


# ------------------------------------------------------------- the definitions, in 64 bits

def _plan_exact(case, seed):
    s = prepare(case, seed)
    bs = case["block"]
    new, old = _plan_lengths(case)
    tables, free, n = s["tables"].tolist(), s["free"].tolist(), s["tokens"]
    slots, where, req, used = [-1] * n, [0] * n, [-1] * n, 0
    at = _starts(new)
    for r, (k, p) in enumerate(zip(new, old)):
        for i in range(k):
            if p % bs == 0:
                tables[r][p // bs] = free[used]
                used += 1
            slots[at[r] + i], where[at[r] + i], req[at[r] + i] = tables[r][p // bs] * bs + p % bs, p, r
            p += 1
    return dict(query_start_loc=_ints(at), seq_lens=_ints([a + b for a, b in zip(new, old)]),
                slot_mapping=_ints(slots, I64), positions=_ints(where, I64), token_request=_ints(req),
                blocks_used=_ints([used]), block_tables=_ints(tables))


def _groups_exact(case, seed):
    s = prepare(case, seed)
    n, bs, tables, lens = case["requests"], case["block"], s["tables"].tolist(), s["lens"].tolist()
    starts, shared = [0], [0]
    for r in range(1, n):
        k = 0
        while k < min(lens[r - 1], lens[r]) // bs and tables[r - 1][k] == tables[r][k]:
            k += 1
        if k * bs >= case["least"]:
            shared[-1] = min(shared[-1], k * bs) if starts[-1] < r - 1 else k * bs
        else:
            starts.append(r)
            shared.append(0)
    return dict(group_start_loc=_ints(starts + [n] * (n + 1 - len(starts))),
                shared_lens=_ints(shared + [0] * (n - len(shared))))


def exact(case, seed):
    if case["kind"] == "plan":
        return _plan_exact(case, seed)
    if case["kind"] == "groups":
        return _groups_exact(case, seed)
    s, kc, vc = _make(case, seed)
    new, lens = _attn_lengths(case)
    pre, at, g = _prefix_lens(case, new, lens), _starts(new), case["hq"] // case["hkv"]
    f64 = torch.float64
    q, rk, rv = s["q"].to(f64), s["rk"].to(f64), s["rv"].to(f64)
    out = torch.zeros(q.shape, dtype=f64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=f64, device=DEV)
    for b, (k, t) in enumerate(zip(new, lens)):
        blocks = s["tables"][b, : -(-t // case["block"])].long()
        p, j = torch.arange(t - k, t, device=DEV)[:, None], torch.arange(t, device=DEV)[None, :]
        seen = j <= p
        if pre is not None:
            seen = seen | (j < pre[b])
        if case["window"]:
            seen = seen & (j > p - case["window"])
        if case["docs"]:
            seen = seen & (j >= p // case["docs"] * case["docs"])
        for head in range(case["hkv"]):
            key = s["kcen"].to(f64)[kc[blocks, head].reshape(-1, D)[:t].long()] @ rk
            key = key * s["kn"][blocks, head].reshape(-1, 1)[:t].to(f64)
            val = s["vcen"].to(f64)[vc[blocks, head].reshape(-1, D)[:t].long()] @ rv
            val = val * s["vn"][blocks, head].reshape(-1, 1)[:t].to(f64)
            for hh in range(head * g, head * g + g):
                x = q[at[b]: at[b + 1], hh] @ key.t() / math.sqrt(D)
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if case["alibi"]:
                    x = x - s["slopes"][hh].to(f64) * (p - j)
                x = x.masked_fill(~seen, -math.inf)
                l = torch.logsumexp(x, -1)
                lse[at[b]: at[b + 1], hh] = l
                out[at[b]: at[b + 1], hh] = torch.exp(x - l[:, None]) @ val
    return [out, lse] if case["lse"] else [out]
