"""No-GPU checks at the edges of the attention half of a step: frequencies over long trained contexts, refusals."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from lattice_b200 import KvCache, _lib, rope_frequencies
from lattice_b200._lib import KvAppendArgs, KvCacheDesc, TreeAttentionArgs


def yarn_by_definition(rot, theta, factor, original_len, fast, slow):
    """Peng et al. 2023: a ramp over the pair index between the pairs that turn `fast` and `slow` times in original_len
    positions, rounded outwards to whole pairs and kept within the channels of a head."""
    pair = lambda turns: rot * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
    out = []
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        share = 1 - min(max((i - low) / (high - low), 0), 1)                  # of the unscaled frequency
        out.append(f / factor * (1 - share) + f * share)
    return np.array(out)


@pytest.mark.parametrize("rot, theta, original_len, slow", [
    (128, 1e4, 4096, 1.0), (128, 1e4, 65536, 1.0), (128, 1e4, 131072, 1.0), (64, 1e4, 1 << 20, 1.0), (64, 1e4, 131072, 4.0), (2, 1e4, 131072, 1.0),
    (96, 500000.0, 1 << 24, 1.0), (128, 10.0, 100.0, 1.0),
])
def test_yarn_where_the_slowest_pair_still_turns(rot, theta, original_len, slow):
    """Beyond about 2 pi theta trained positions the pair that turns `slow` times lies behind the last one: the last pairs
    are on the ramp, not at its end."""
    f, _ = rope_frequencies(rot, theta, "yarn", factor=4.0, original_len=original_len, beta_fast=32.0, beta_slow=slow)
    np.testing.assert_allclose(f, yarn_by_definition(rot, theta, 4.0, original_len, 32.0, slow), rtol=1e-12)
    plain = np.array([theta ** (-2 * i / rot) for i in range(rot // 2)])
    turns = plain * original_len / (2 * math.pi)
    assert np.all(f[turns > slow] > plain[turns > slow] / 4 * (1 + 1e-9))     # what turns more often keeps a share


@pytest.mark.parametrize("original_len", [1.0, 4.0, 6.0])
def test_yarn_where_no_pair_turns(original_len):
    """A context so short that even the fastest pair turns less than beta_slow times: all of them are interpolated."""
    f, _ = rope_frequencies(64, 1e4, "yarn", factor=4.0, original_len=original_len)
    np.testing.assert_allclose(f, [1e4 ** (-2 * i / 64) / 4 for i in range(32)], rtol=1e-12)


# ---- arguments -----------------------------------------------------------------------------------------------------

P = 0x10000          # a made-up device address, 16-byte aligned: refused calls never touch it


@pytest.fixture(scope="module")
def L():
    from lattice_b200 import build as lq4_build
    lq4_build.build()
    return _lib.lib()


def cache_desc():
    return KvCacheDesc(k=P, v=P, pages=8, page_size=16, kv_heads=2, head_dim=64, page_table=P, batch=2, max_pages=4)


def test_append_of_no_rows_checks_what_it_reads(L):
    """Without rows k and v are not read, the lengths are where new_lens is asked for."""
    def call(**change):
        fields = dict(cache=C.pointer(cache_desc()), k=None, v=None, dtype=1, rows=0, kv_lens=P, new_lens=2 * P)
        fields.update(change)
        return L.lq4_kv_append(None, C.byref(KvAppendArgs(**fields)), None), L.lq4_last_error()
    assert call() == (_lib.ERR_NULL, b"ctx is NULL")
    assert call(kv_lens=None, new_lens=None) == (_lib.ERR_NULL, b"ctx is NULL")
    status, text = call(kv_lens=None)
    assert status == _lib.ERR_NULL and b"kv_lens" in text
    assert call(new_lens=P + 2)[0] == _lib.ERR_ALIGN


def test_every_thread_packs_its_own_arguments():
    """The library reads packed arguments while another thread may run, and pack its own."""
    from concurrent.futures import ThreadPoolExecutor
    from lattice_b200.backend import _ArgumentBuffer
    args = _ArgumentBuffer()
    args.buf[0:4] = b"here"
    with ThreadPoolExecutor(1) as pool:
        there = pool.submit(lambda: (args.at, args.buf[0:4])).result()
    assert there[0] != args.at and there[1] == bytes(4)
    assert args.buf[0:4] == b"here" and args.at == C.addressof(args.buf)


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_a_cache_of_expanded_tensors_is_refused(dim):
    """A stride of 0 means dense to the library, which would then read and write behind an expanded tensor."""
    shape, small = [4, 8, 2, 16], [4, 8, 2, 16]
    small[dim] = 1
    k = torch.zeros(small, dtype=torch.bfloat16).expand(shape)
    with pytest.raises(ValueError, match="expanded"):
        KvCache(k, k.clone().as_strided(shape, k.stride()), torch.zeros(1, 2, dtype=torch.int32))


def test_strides_of_single_entries_do_not_count(monkeypatch):
    """The stride of a dimension of one entry may be anything."""
    x = torch.zeros(1000, dtype=torch.bfloat16).as_strided((1, 4, 1, 16), (3, 16, 5, 1))
    table = torch.zeros(1, 1, dtype=torch.int32)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)          # as if they lay on a GPU; nothing is launched
    cache = KvCache(x, x, table)
    assert (cache.desc.page_stride, cache.desc.slot_stride, cache.desc.head_stride) == (0, 16, 0)


@pytest.mark.parametrize("scale, ok", [(3e38, False), (-3e38, False), (2.3e38, True), (-2.3e38, True), (0.0, True)])
def test_attention_refuses_scales_that_overflow(L, scale, ok):
    """The kernels work in units of log2: scale times log2(e) has to be finite as well."""
    a = TreeAttentionArgs(q=P, out=2 * P, dtype=1, k=P, v=P, nodes=3, q_heads=4, q_batch=768, q_node=256, q_head=64, out_batch=768, out_node=256,
                          out_head=64, kv_batch=384, kv_node=128, kv_head=64, kv_lens=P, scale=scale, cache=C.pointer(cache_desc()))
    assert L.lq4_tree_attention(None, C.byref(a), None) == (_lib.ERR_NULL if ok else _lib.ERR_SHAPE)      # (in order: only the context is missing)


def test_the_status_is_read_on_the_backends_device(monkeypatch):
    """Whichever device is current: the calls ran on the current stream of the backend's."""
    from types import SimpleNamespace
    from lattice_b200 import backend
    seen = []
    monkeypatch.setattr(backend, "_raw_stream", lambda device: 1000 + device)
    monkeypatch.setattr(backend, "_stream", lambda: 1)
    monkeypatch.setattr(backend._lib, "lib", lambda: SimpleNamespace(lq4_ctx_check=lambda ctx, stream: seen.append((ctx, stream)) or 0))
    be = backend.CudaQ4Backend.__new__(backend.CudaQ4Backend)
    be._ctx, be.device = 77, 3
    be.check_device_status()
    be._ctx = None                                                           # (nothing to destroy)
    assert seen == [(77, 1003)]
