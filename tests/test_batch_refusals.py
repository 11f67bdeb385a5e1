"""Refusals of the batch operators' C entry points: each call is wrong in one argument and is turned
down before anything is launched, so no GPU is needed."""

import ctypes

import pytest

import capi
from turboquant_kv.vllm_plugin import AttentionVariant

ADDR = 1 << 20  # an aligned address that no refused call looks at
i32, i64, f32, ptr, size = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t


class Variant(ctypes.Structure):
    _fields_ = [("softcap", f32), ("alibi_slopes", ptr), ("window", i32), ("prefix_lens", ptr), ("token_starts", ptr)]


ATTENTION = [("q", ptr, ADDR), ("dtype", i32, 0), ("n_tokens", i32, 3), ("q_stride", i64, 512), ("hq", i32, 8), ("hkv", i32, 2),
             ("d", i32, 64), ("kpairs", ptr, ADDR), ("knorm", ptr, ADDR), ("vtile", ptr, ADDR), ("vnorm", ptr, ADDR),
             ("num_blocks", i64, 4), ("block_size", i32, 16), ("vbits", i32, 2), ("block_tables", ptr, ADDR),
             ("table_stride", i64, 2), ("max_blocks", i32, 2), ("query_start_loc", ptr, ADDR), ("seq_lens", ptr, ADDR),
             ("n_seqs", i32, 1), ("group_start_loc", ptr, ADDR), ("shared_lens", ptr, ADDR), ("n_groups", i32, 1),
             ("kcentroids", ptr, ADDR), ("vcentroids", ptr, ADDR), ("krotation", ptr, ADDR), ("vrotation", ptr, ADDR),
             ("transposed", i32, 0), ("scale", f32, 0.125), ("variant", ptr, None), ("out", ptr, ADDR), ("out_stride", i64, 512),
             ("zero_tail", i32, 0), ("lse", ptr, None), ("workspace", ptr, ADDR), ("workspace_bytes", size, 0),
             ("stream", ptr, None)]
PLAN = [("new_lens", ptr, ADDR), ("context_lens", ptr, ADDR), ("n_requests", i32, 2), ("block_tables", ptr, ADDR),
        ("table_stride", i64, 3), ("max_blocks", i32, 3), ("free_blocks", ptr, ADDR), ("n_free", i64, 4),
        ("free_start", ptr, None), ("block_size", i32, 16), ("n_tokens", i32, 5), ("query_start_loc", ptr, ADDR),
        ("seq_lens", ptr, ADDR), ("slot_mapping", ptr, ADDR), ("positions", ptr, ADDR), ("token_request", ptr, ADDR),
        ("blocks_used", ptr, ADDR), ("stream", ptr, None)]
GROUPS = [("block_tables", ptr, ADDR), ("table_stride", i64, 3), ("max_blocks", i32, 3), ("context_lens", ptr, ADDR),
          ("n_requests", i32, 2), ("block_size", i32, 16), ("min_tokens", i32, 16), ("group_start_loc", ptr, ADDR),
          ("shared_lens", ptr, ADDR), ("workspace", ptr, ADDR), ("workspace_bytes", size, 0), ("stream", ptr, None)]


def refused(name, spec, changed):
    lib = capi.lib()
    fn = getattr(lib, name)
    fn.argtypes, fn.restype = [t for _, t, _ in spec], i32
    assert set(changed) <= {n for n, _, _ in spec}
    assert fn(*[changed.get(n, v) for n, _, v in spec]) != 0
    return lib.tq_last_error().decode()


@pytest.mark.parametrize("changed,why", [
    (dict(dtype=9), "dtype"), (dict(d=128), "head_dim 64"), (dict(vbits=1), "2-4 bit"), (dict(vbits=5), "2-4 bit"),
    (dict(hkv=0), "multiple"), (dict(hq=9), "multiple"), (dict(hq=1), "multiple"), (dict(block_size=8), "power-of-two"),
    (dict(block_size=48), "power-of-two"), (dict(n_tokens=-1), "bad sizes"), (dict(num_blocks=-1), "bad sizes"),
    (dict(n_groups=-1), "bad sizes"), (dict(n_seqs=8193), "8192"), (dict(n_groups=8193), "8192"),
    (dict(num_blocks=2 ** 32), "blocks"), (dict(table_stride=1), "overlap"),
    (dict(max_blocks=2 ** 27, table_stride=2 ** 27), "capacity"), (dict(q_stride=511), "overlap"),
    (dict(out_stride=256), "overlap"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(block_tables=None), "null"),
    (dict(query_start_loc=None), "null"), (dict(seq_lens=None), "null"), (dict(group_start_loc=None), "null"),
    (dict(shared_lens=None), "null"), (dict(kpairs=None), "null"), (dict(vnorm=None), "null"), (dict(kcentroids=None), "null"),
    (dict(vrotation=None), "null"), (dict(q=ADDR + 8), "aligned"), (dict(out=ADDR + 4), "aligned"),
    (dict(vtile=ADDR + 2), "aligned"), (dict(krotation=ADDR + 4), "aligned"), (dict(q_stride=513), "strides"),
    (dict(dtype=1, out_stride=516), "strides"), (dict(n_tokens=2 ** 30, hq=64, hkv=1, q_stride=4096, out_stride=4096), "query rows"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=1000), "workspace")])
def test_attention(changed, why):
    assert why in refused("tq_attention_batch_paged_dl", ATTENTION, changed)


@pytest.mark.parametrize("softcap,window", [(-1.0, 0), (float("inf"), 0), (float("nan"), 0), (1e-38, 0), (2e30, 0), (0.0, -1)])
def test_attention_variant(softcap, window):
    v = Variant(softcap=softcap, window=window)
    why = refused("tq_attention_batch_paged_dl", ATTENTION, dict(variant=ctypes.addressof(v)))
    assert ("window" if window else "softcap") in why


@pytest.mark.parametrize("changed,why", [
    (dict(n_requests=-1), "requests"), (dict(n_requests=8193), "8192"), (dict(block_size=0), "block_size"),
    (dict(n_tokens=-1), "bad sizes"), (dict(n_free=-1), "bad sizes"), (dict(table_stride=2), "overlap"),
    (dict(new_lens=None), "null"), (dict(block_tables=None), "null"), (dict(free_blocks=None), "null"),
    (dict(slot_mapping=None), "null"), (dict(query_start_loc=None), "null"), (dict(blocks_used=None), "null")])
def test_plan(changed, why):
    assert why in refused("tq_paged_batch_plan", PLAN, changed)


@pytest.mark.parametrize("changed,why", [
    (dict(n_requests=-1), "requests"), (dict(n_requests=8193), "8192"), (dict(block_size=0), "block_size"),
    (dict(min_tokens=0), "min_tokens"), (dict(table_stride=2), "overlap"), (dict(max_blocks=2 ** 28, table_stride=2 ** 28), "capacity"),
    (dict(block_tables=None), "null"), (dict(context_lens=None), "null"), (dict(shared_lens=None), "null"),
    (dict(workspace_bytes=4), "workspace")])
def test_groups(changed, why):
    assert why in refused("tq_shared_prefix_groups", GROUPS, changed)


def test_workspaces_of_wrong_sizes_are_empty():
    fn = capi.lib().tq_attention_batch_workspace_bytes
    fn.argtypes, fn.restype = [i32, i32, i32, i32, i32, i32, i64], size
    for n, hq, hkv, B, g, cap in ((0, 8, 2, 1, 0, 64), (3, 8, 3, 1, 0, 64), (3, 8, 0, 1, 0, 64), (3, 8, 2, -1, 0, 64), (3, 8, 2, 1, 0, -1)):
        assert fn(0, n, hq, hkv, B, g, cap) == 0


@pytest.mark.parametrize("kw", [dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(window=-1)])
def test_score_variants(kw):
    with pytest.raises(ValueError):
        AttentionVariant(**kw)
