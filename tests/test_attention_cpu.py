"""No-GPU checks of the attention half of a step: refusals of the C ABI before any device call, the frequencies of
rotary positions, and the argument checks of the Python objects."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from lattice_b200 import KvCache, Lq4Error, RopeTable, _lib, build as lq4_build, rope_frequencies
from lattice_b200._lib import KvAppendArgs, KvCacheDesc, RopeArgs, RopeDesc, RopePart, RopeScaling, TreeAttentionArgs, VerifyArgs


@pytest.fixture(scope="module")
def L():
    lq4_build.build()
    return _lib.lib()


P = 0x10000          # a made-up device address, 16-byte aligned: refused calls never touch it


def rope_args(n_parts=1, rows=4, head_dim=64, rot=64, layout=0, scale=1.0, freq=P, positions=P, rope=True, **part):
    fields = dict(x=P, out=2 * P, x_dtype=0, out_dtype=0, heads=2, turn=1, x_row=128, x_head=64, out_row=128, out_head=64)
    fields.update(part)
    arr = (RopePart * max(n_parts, 1))(*[RopePart(**fields) for _ in range(max(n_parts, 1))])
    desc = RopeDesc(freq, rot, layout, scale)
    return RopeArgs(arr, n_parts, rows, head_dim, positions, C.pointer(desc) if rope else None)


@pytest.mark.parametrize("change, status", [
    (dict(), _lib.ERR_NULL),                                    # everything in order: only the context is missing
    (dict(n_parts=5), _lib.ERR_SHAPE),
    (dict(head_dim=0), _lib.ERR_SHAPE),
    (dict(head_dim=1025), _lib.ERR_SHAPE),
    (dict(heads=4097), _lib.ERR_SHAPE),
    (dict(rows=1 << 31), _lib.ERR_OVERFLOW),
    (dict(x_row=1 << 59), _lib.ERR_OVERFLOW),
    (dict(x_dtype=2), _lib.ERR_DTYPE),
    (dict(out_dtype=7), _lib.ERR_DTYPE),
    (dict(turn=2), _lib.ERR_ROT),
    (dict(rot=63), _lib.ERR_ROT),
    (dict(rot=0), _lib.ERR_ROT),
    (dict(rot=66), _lib.ERR_ROT),
    (dict(layout=2), _lib.ERR_ROT),
    (dict(scale=math.nan), _lib.ERR_ROT),
    (dict(scale=math.inf), _lib.ERR_ROT),
    (dict(x=None), _lib.ERR_NULL),
    (dict(out=None), _lib.ERR_NULL),
    (dict(freq=None), _lib.ERR_NULL),
    (dict(positions=None), _lib.ERR_NULL),
    (dict(rope=False), _lib.ERR_NULL),
    (dict(x=P + 2), _lib.ERR_ALIGN),
    (dict(x_dtype=1, x=P + 1), _lib.ERR_ALIGN),
    (dict(freq=P + 4), _lib.ERR_ALIGN),
    (dict(out=P, out_row=256), _lib.ERR_SHAPE),                 # in place with another stride
    (dict(out=P, out_dtype=1), _lib.ERR_SHAPE),                 # in place with another type
])
def test_rope_refusals(L, change, status):
    a = rope_args(**change)
    assert L.lq4_rope_rows(None, C.byref(a), None) == status
    assert status != _lib.ERR_NULL or b"ctx" in L.lq4_last_error() or change


def cache_desc(**change):
    fields = dict(k=P, v=P, pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=0, slot_stride=0, head_stride=0,
                  page_table=P, batch=2, max_pages=4)
    fields.update(change)
    return KvCacheDesc(**fields)


CACHE_REFUSALS = [
    (dict(head_dim=0), _lib.ERR_SHAPE), (dict(head_dim=12), _lib.ERR_SHAPE), (dict(head_dim=264), _lib.ERR_SHAPE),
    (dict(kv_heads=0), _lib.ERR_SHAPE), (dict(kv_heads=5000), _lib.ERR_SHAPE), (dict(page_size=0), _lib.ERR_SHAPE),
    (dict(pages=1 << 31), _lib.ERR_OVERFLOW), (dict(max_pages=1 << 28), _lib.ERR_OVERFLOW),
    (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL), (dict(page_table=None), _lib.ERR_NULL),
    (dict(k=P + 8), _lib.ERR_ALIGN), (dict(v=P + 2), _lib.ERR_ALIGN), (dict(page_table=P + 2), _lib.ERR_ALIGN),
    (dict(page_stride=4), _lib.ERR_ALIGN), (dict(slot_stride=12), _lib.ERR_ALIGN), (dict(head_stride=1), _lib.ERR_ALIGN),
]


def append_args(cache=None, **change):
    fields = dict(k=P, v=P, dtype=1, rows=3, batch_stride=384, row_stride=128, head_stride=64, kv_lens=P, counts=None, index=None, new_lens=2 * P)
    fields.update(change)
    return KvAppendArgs(C.pointer(cache if cache is not None else cache_desc()), *[fields[n] for n, _ in KvAppendArgs._fields_[1:]])


@pytest.mark.parametrize("change, status", CACHE_REFUSALS)
def test_append_refuses_bad_caches(L, change, status):
    a = append_args(cache_desc(**change))
    assert L.lq4_kv_append(None, C.byref(a), None) == status


@pytest.mark.parametrize("change, status", [
    (dict(), _lib.ERR_NULL), (dict(dtype=2), _lib.ERR_DTYPE), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL),
    (dict(kv_lens=None), _lib.ERR_NULL), (dict(k=P + 2), _lib.ERR_ALIGN), (dict(row_stride=4), _lib.ERR_ALIGN),
    (dict(batch_stride=1), _lib.ERR_ALIGN), (dict(head_stride=63), _lib.ERR_ALIGN), (dict(index=P + 1), _lib.ERR_ALIGN),
    (dict(new_lens=P), _lib.ERR_SHAPE), (dict(rows=1 << 31), _lib.ERR_OVERFLOW), (dict(row_stride=1 << 59), _lib.ERR_OVERFLOW),
])
def test_append_refusals(L, change, status):
    a = append_args(**change)
    assert L.lq4_kv_append(None, C.byref(a), None) == status
    assert L.lq4_kv_append(None, None, None) == _lib.ERR_NULL


def turns_left(f, n):                     # turns of frequency f in n positions
    return f * n / (2 * math.pi)


@pytest.mark.parametrize("rot", [2, 6, 64, 128, 250])
def test_frequencies_plain_linear_ntk(rot):
    half = rot // 2
    base = np.array([10000.0 ** (-2.0 * i / rot) for i in range(half)])
    f, s = rope_frequencies(rot, 10000.0)
    np.testing.assert_allclose(f[:half], base, rtol=1e-14)
    assert s == 1.0
    f, s = rope_frequencies(rot, 10000.0, "linear", factor=8.0)
    np.testing.assert_allclose(f[:half], base / 8, rtol=1e-14)
    if rot > 2:
        f, s = rope_frequencies(rot, 10000.0, "ntk", factor=8.0)
        assert s == 1.0 and f[0] == 1.0
        np.testing.assert_allclose(f[half - 1], base[-1] / 8, rtol=1e-12)      # the slowest pair as interpolated


@pytest.mark.parametrize("kind", ["yarn", "bands"])
@pytest.mark.parametrize("rot", [64, 128])
def test_frequencies_ramped(kind, rot):
    half, factor, n = rot // 2, 4.0, 4096.0
    plain, _ = rope_frequencies(rot, 1e6)
    f, s = rope_frequencies(rot, 1e6, kind, factor=factor, original_len=n, beta_fast=32.0, beta_slow=1.0)
    assert s == pytest.approx(0.1 * math.log(4) + 1 if kind == "yarn" else 1.0, rel=1e-6)
    share = (f / plain - 1 / factor) / (1 - 1 / factor)                        # of the unscaled frequency
    assert np.all(np.diff(share) <= 1e-12) and share[0] == pytest.approx(1.0)
    for i in range(half):
        t = turns_left(plain[i], n)
        if kind == "bands":
            assert share[i] == pytest.approx(min(max((t - 1) / 31, 0), 1), abs=1e-9)
        elif t >= 32 * 1e6 ** (1 / half):                                      # a pair beyond the rounded border
            assert share[i] == pytest.approx(1.0)
        elif t <= 1 / 1e6 ** (1 / half):
            assert share[i] == pytest.approx(0.0, abs=1e-12)


@pytest.mark.parametrize("change", [dict(kind=9), dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=2, kind=2), dict(theta=1.0), dict(theta=math.inf),
                                    dict(factor=0.5), dict(factor=math.nan), dict(kind=3, beta_fast=1.0), dict(kind=4, beta_slow=0.0),
                                    dict(kind=3, original_len=0.0)])
def test_frequency_refusals(L, change):
    fields = dict(kind=1, rot_dim=64, theta=1e4, factor=2.0, original_len=4096.0, beta_fast=32.0, beta_slow=1.0)
    fields.update(change)
    freq, scale = np.zeros(64), C.c_float()
    assert L.lq4_rope_frequencies(C.byref(RopeScaling(**fields)), freq.ctypes.data, C.byref(scale)) == _lib.ERR_ROT
    assert not freq.any()


def test_python_objects_refuse():
    with pytest.raises(ValueError):
        rope_frequencies(64, scaling="other")
    with pytest.raises(Lq4Error):
        rope_frequencies(7)
    with pytest.raises(TypeError):
        RopeTable(torch.ones(4))                                               # float32
    with pytest.raises(ValueError):
        RopeTable(torch.ones(4, dtype=torch.float64), layout="thirds")
    k = torch.zeros(2, 4, 1, 8, dtype=torch.bfloat16)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(TypeError):
        KvCache(k.float(), k.float(), table)
    with pytest.raises(TypeError):
        KvCache(k, k, table.long())
    with pytest.raises(ValueError):
        KvCache(k, k[:, :2], table)
    with pytest.raises(ValueError):
        KvCache(k, k.clone(), table)                                           # not on a GPU


def attend_args(cache=None, **change):
    fields = dict(q=P, out=2 * P, dtype=1, k=P, v=P, nodes=3, q_heads=4, q_batch=768, q_node=256, q_head=64, out_batch=768, out_node=256,
                  out_head=64, kv_batch=384, kv_node=128, kv_head=64, kv_lens=P, node_counts=None, parents=None, scale=0.125)
    fields.update(change)
    return TreeAttentionArgs(cache=C.pointer(cache if cache is not None else cache_desc()), **fields)


@pytest.mark.parametrize("change, status", CACHE_REFUSALS)
def test_attention_refuses_bad_caches(L, change, status):
    a = attend_args(cache_desc(**change))
    assert L.lq4_tree_attention(None, C.byref(a), None) == status


@pytest.mark.parametrize("change, status", [
    (dict(), _lib.ERR_NULL), (dict(dtype=2), _lib.ERR_DTYPE), (dict(nodes=65), _lib.ERR_SHAPE), (dict(q_heads=0), _lib.ERR_SHAPE),
    (dict(q_heads=5), _lib.ERR_SHAPE), (dict(q_heads=2 * 1025), _lib.ERR_SHAPE), (dict(scale=math.inf), _lib.ERR_SHAPE), (dict(scale=math.nan), _lib.ERR_SHAPE),
    (dict(q=None), _lib.ERR_NULL), (dict(out=None), _lib.ERR_NULL), (dict(k=None), _lib.ERR_NULL), (dict(v=None), _lib.ERR_NULL),
    (dict(kv_lens=None), _lib.ERR_NULL), (dict(q=P + 1), _lib.ERR_ALIGN), (dict(dtype=0, out=P + 2), _lib.ERR_ALIGN), (dict(k=P + 8), _lib.ERR_ALIGN),
    (dict(kv_node=4), _lib.ERR_ALIGN), (dict(kv_head=2), _lib.ERR_ALIGN), (dict(kv_batch=1), _lib.ERR_ALIGN), (dict(parents=P + 2), _lib.ERR_ALIGN),
    (dict(q_batch=1 << 58), _lib.ERR_OVERFLOW), (dict(out_head=1 << 41), _lib.ERR_OVERFLOW),
])
def test_attention_refusals(L, change, status):
    a = attend_args(**change)
    assert L.lq4_tree_attention(None, C.byref(a), None) == status
    assert L.lq4_tree_attention(None, None, None) == _lib.ERR_NULL


def verify_args(**change):
    fields = dict(target_logits=P, draft_logits=P, dtype=0, batch=2, nodes=4, vocab=100, target_batch=400, target_node=100, draft_batch=400,
                  draft_node=100, tokens=P, parents=P, node_counts=P, uniforms=P, temperature=P, path=P, path_len=P, next_token=P)
    fields.update(change)
    return VerifyArgs(**fields)


@pytest.mark.parametrize("change, status", [
    (dict(), _lib.ERR_NULL), (dict(dtype=2), _lib.ERR_DTYPE), (dict(nodes=0), _lib.ERR_SHAPE), (dict(nodes=65), _lib.ERR_SHAPE),
    (dict(vocab=0), _lib.ERR_SHAPE), (dict(vocab=1 << 30), _lib.ERR_OVERFLOW), (dict(batch=1 << 26), _lib.ERR_OVERFLOW),
    (dict(target_batch=1 << 60), _lib.ERR_OVERFLOW), (dict(draft_node=1 << 53), _lib.ERR_OVERFLOW),
    (dict(target_logits=None), _lib.ERR_NULL), (dict(tokens=None), _lib.ERR_NULL), (dict(uniforms=None), _lib.ERR_NULL), (dict(path=None), _lib.ERR_NULL),
    (dict(path_len=None), _lib.ERR_NULL), (dict(next_token=None), _lib.ERR_NULL), (dict(target_logits=P + 2), _lib.ERR_ALIGN),
    (dict(draft_logits=P + 1, dtype=1), _lib.ERR_ALIGN), (dict(uniforms=P + 2), _lib.ERR_ALIGN), (dict(path=P + 1), _lib.ERR_ALIGN),
])
def test_verify_refusals(L, change, status):
    a = verify_args(**change)
    assert L.lq4_verify_draft(None, C.byref(a), None) == status
    assert L.lq4_verify_draft(None, None, None) == _lib.ERR_NULL


def test_packed_arguments_match_the_structures():
    from lattice_b200.backend import CudaQ4Backend as B
    for packer, desc in ((B._ROPE_PART, RopePart), (B._ROPE_ARGS, RopeArgs), (B._APPEND_ARGS, KvAppendArgs), (B._TREE_ARGS, TreeAttentionArgs),
                         (B._VERIFY_ARGS, VerifyArgs)):
        buf = C.create_string_buffer(C.sizeof(desc))
        values = list(range(1, len(packer.unpack(bytes(packer.size))) + 1))
        packer.pack_into(buf, 0, *values)
        got = desc.from_buffer(buf)
        flat = [C.cast(v, C.c_void_p).value if hasattr(v, "contents") else v for v in (getattr(got, n) for n, _ in desc._fields_)]
        assert flat == values and -(-packer.size // 8) * 8 == C.sizeof(desc)
