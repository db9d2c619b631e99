"""Rotary positions, cache append, tree attention and draft verification on the GPU, against plain 64-bit implementations."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def be():
    from lattice_b200 import CudaQ4Backend
    b = CudaQ4Backend(0)
    yield b
    b.close()


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(seed, *shape):
    return torch.randn(*shape, generator=rng(seed), dtype=torch.float64)


def on_gpu(x, dtype):
    return x.to(dtype).cuda()


# ---- rotary positions ----------------------------------------------------------------------------------------------

def rope_ref(x, pos, freq, layout, scale, turn):
    """64-bit rotation of [rows, heads, dim], and per element the sum of the magnitudes that met in it."""
    x = x.double()
    if turn == 0:
        return x, torch.zeros_like(x)
    a = pos.double()[:, None] * torch.from_numpy(freq)
    c, s = (a.cos() * scale)[:, None], (a.sin() * scale * turn)[:, None]
    r = 2 * freq.size
    at = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., at[0]] = x[..., at[0]] * c - x[..., at[1]] * s
    y[..., at[1]] = x[..., at[0]] * s + x[..., at[1]] * c
    mag[..., at[0]] = mag[..., at[1]] = (x[..., at[0]].abs() + x[..., at[1]].abs()) * abs(scale)
    return y, mag


def assert_rope(got, ref, mag):
    # The remainder of the angle in f32: half a step of 2^-25 turns, 2 pi 2^-26 rad; sincospi: a step of at most 2^-24;
    # scale, two products and a sum: 4 roundings of 2^-24.  Together under 4.0e-7 of the magnitudes; then the store.
    tol = 4.0e-7 * mag + HALF_STEP[got.dtype] * ref.abs() * (1 + 1e-6) + 1e-30
    assert bool(((got.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows, heads, dim, rot, src, dst", [
    (1, 1, 8, 2, F32, F32), (1, 40, 128, 128, F32, BF16), (3, 5, 80, 20, BF16, F32), (7, 2, 130, 6, F32, F32), (257, 3, 64, 64, BF16, BF16),
    (33, 24, 256, 64, BF16, BF16), (2, 1, 1024, 1024, F32, F32), (1000, 1, 6, 4, F32, BF16), (5, 3, 72, 16, BF16, BF16),
])
def test_rope_against_64_bits(be, layout, rows, heads, dim, rot, src, dst):
    from lattice_b200 import RopeTable, rope_frequencies
    freq, scale = rope_frequencies(rot, 1e6, "yarn", factor=4.0) if rot > 2 else rope_frequencies(rot, 1e6)
    freq = freq[:rot // 2]
    x = normal(1, rows, heads, dim).to(src)
    pos = torch.randint(-5, 2 ** 20, (rows,), generator=rng(2), dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    table = RopeTable(torch.from_numpy(freq).cuda(), layout, scale)
    for turn in (1, -1, 0):
        y, = be.rope_rows([(x.cuda(), turn)], pos.cuda(), table, out_dtype=dst)
        assert y.dtype == dst
        assert_rope(y, *rope_ref(x, pos, freq, layout, np.float32(scale), turn))


def test_rope_fused_row_in_one_launch_and_in_place(be):
    from lattice_b200 import RopeTable
    rows, hq, hk, dim = 19, 10, 2, 128
    fused = normal(3, rows, (hq + 2 * hk) * dim).float()
    table = RopeTable.from_config(128, "cuda", theta=1e6)
    freq = table.freq.cpu().numpy()
    pos = torch.arange(100, 100 + rows, dtype=torch.int32)
    g = fused.cuda().view(rows, hq + 2 * hk, dim)
    q, k, v = g.split([hq, hk, hk], 1)
    before = be.launch_count
    outs = be.rope_rows([(q, 1), (k, 1), (v, 0)], pos.cuda(), table, out_dtype=BF16)
    assert be.launch_count == before + 1
    cpu = fused.view(rows, hq + 2 * hk, dim).split([hq, hk, hk], 1)
    for y, x, turn in zip(outs, cpu, (1, 1, 0)):
        assert_rope(y, *rope_ref(x, pos, freq, "half", 1.0, turn))
    be.rope_rows([(q, 1), (k, -1)], pos.cuda(), table, outs=[q, k])             # in place, strided
    assert_rope(q, *rope_ref(cpu[0], pos, freq, "half", 1.0, 1))
    assert_rope(k, *rope_ref(cpu[1], pos, freq, "half", 1.0, -1))
    assert torch.equal(v.cpu(), cpu[2])                                         # what is not named stays as it was


def test_rope_unaligned_rows(be):
    """Offsets and strides that no vector fits."""
    from lattice_b200 import RopeTable
    table = RopeTable.from_config(32, "cuda", "interleaved")
    flat = normal(4, 5 * 333 + 1).float().cuda()
    x = torch.as_strided(flat, (5, 3, 64), (333, 65, 1), 1)
    pos = torch.arange(5, dtype=torch.int32)
    y, = be.rope_rows([(x, 1)], pos.cuda(), table)
    assert_rope(y, *rope_ref(x.cpu(), pos, table.freq.cpu().numpy(), "interleaved", 1.0, 1))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_transpose_is_the_gradient(be, layout):
    """<turn(x), g> = <x, turn_back(g)> (the formula's gradient), and against differences of a weighted sum."""
    from lattice_b200 import RopeTable
    table = RopeTable.from_config(48, "cuda", layout, scaling="yarn", factor=2.0)
    pos = torch.tensor([0, 3, 70001, 12], dtype=torch.int32).cuda()
    x, g = normal(5, 4, 2, 64).float().cuda(), normal(6, 4, 2, 64).float().cuda()
    y, = be.rope_rows([(x, 1)], pos, table)
    back, = be.rope_rows([(g, -1)], pos, table)
    a, b = (y.double() * g.double()).sum(), (x.double() * back.double()).sum()
    # each side is a sum of 512 products whose factors are off by at most 4e-7 of two magnitudes
    assert abs(a - b) <= 2 * 4.0e-7 * 2 * float((x.abs().double().amax() * g.abs().double()).sum())
    d = torch.zeros_like(x)
    d[2, 1, 5] = 0.5
    up, = be.rope_rows([(x + d, 1)], pos, table)
    down, = be.rope_rows([(x - d, 1)], pos, table)
    slope = float(((up.double() - down.double()) * g.double()).sum())           # linear: exact but for rounding
    assert slope == pytest.approx(float(back[2, 1, 5]), abs=1e-4)


def test_rope_empty_and_other_stream(be):
    from lattice_b200 import RopeTable
    table = RopeTable.from_config(16, "cuda")
    assert be.rope_rows([], torch.zeros(0, dtype=torch.int32).cuda(), table) == []
    y, = be.rope_rows([(torch.zeros(0, 3, 16).cuda(), 1)], torch.zeros(0, dtype=torch.int32).cuda(), table)
    assert y.shape == (0, 3, 16)
    x, pos = normal(7, 9, 3, 16).float(), torch.arange(9, dtype=torch.int32)
    side = torch.cuda.Stream()
    xg, pg = x.cuda(), pos.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, = be.rope_rows([(xg, 1)], pg, table)
    side.synchronize()
    assert_rope(y, *rope_ref(x, pos, table.freq.cpu().numpy(), "half", 1.0, 1))


# ---- cache append --------------------------------------------------------------------------------------------------

def make_cache(batch, max_pages, page, heads, dim, seed=10, order="dense", spare=3):
    """A cache of known contents with shuffled pages; `order` "heads" keeps [pages, heads, page, dim] in memory."""
    from lattice_b200 import KvCache
    pages = batch * max_pages + spare
    table = torch.randperm(pages, generator=rng(seed))[:batch * max_pages].view(batch, max_pages).to(torch.int32)
    kv = []
    for i in range(2):
        x = normal(seed + 1 + i, pages, page, heads, dim).to(BF16)
        kv.append(x.cuda() if order == "dense" else x.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3))
    return KvCache(kv[0], kv[1], table.cuda())


def append_ref(cache, k, v, lens, counts, index):
    """Where the rows land, in plain loops; returns the expected contents and lengths."""
    out = [cache.k.cpu().clone(), cache.v.cpu().clone()]
    table, page = cache.page_table.cpu(), cache.k.shape[1]
    new = []
    for b, n in enumerate(lens):
        c = k.shape[1] if counts is None else counts[b]
        c = 0 if n < 0 else max(c, 0)
        for j in range(c):
            s = n + j
            if s >= table.shape[1] * page:
                continue
            src = j if index is None else index[b][j]
            for o, x in zip(out, (k, v)):
                o[table[b, s // page], s % page] = x[b, src].to(BF16)
        new.append(n if n < 0 else min(n + c, table.shape[1] * page))
    return out[0], out[1], new


def check_append(be, cache, k, v, lens, counts=None, index=None):
    ref = append_ref(cache, k.cpu(), v.cpu(), lens, counts, index)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    new = be.kv_append(cache, k, v, i32(lens), counts=i32(counts), index=i32(index))
    assert torch.equal(cache.k.cpu(), ref[0]) and torch.equal(cache.v.cpu(), ref[1])      # all pages, the untouched ones too
    assert new.tolist() == ref[2]


@pytest.mark.parametrize("order", ["dense", "heads"])
@pytest.mark.parametrize("page, heads, dim, src", [(1, 1, 8, F32), (5, 2, 80, BF16), (16, 8, 128, F32), (64, 3, 256, BF16)])
def test_append_all_rows(be, order, page, heads, dim, src):
    cache = make_cache(3, 40 if page < 16 else 6, page, heads, dim, order=order)
    fused = on_gpu(normal(20, 3, 11, 2 * heads, dim), src)
    check_append(be, cache, fused[:, :, :heads], fused[:, :, heads:], [0, page, 2 * page - 1])
    be.check_device_status()


def test_append_selected_rows(be):
    cache = make_cache(5, 4, 7, 2, 64)
    k, v = on_gpu(normal(21, 5, 6, 2, 64), BF16), on_gpu(normal(22, 5, 6, 2, 64), BF16)
    index = [[0, 2, 5, -1, -1, -1], [0, 1, 2, 3, 4, 5], [3, 3, 3, -1, -1, -1], [-1] * 6, [0, 4, -1, -1, -1, -1]]
    check_append(be, cache, k, v, [0, 13, 6, 9, -1], [3, 6, 3, 0, 2], index)    # the last sequence is left alone
    be.check_device_status()


def test_append_reports_what_it_skips(be):
    from lattice_b200 import Lq4Error
    k = on_gpu(normal(23, 1, 4, 1, 16), BF16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    for lens, counts, index, bad_page in ([6], None, None, False), ([0], [9], None, False), ([0], [2], [[0, 4, 0, 0]], False), \
            ([0], [1], [[-1, 0, 0, 0]], False), ([0], None, None, True):
        cache = make_cache(1, 2, 4, 1, 16)
        if bad_page:
            cache.page_table.fill_(10 ** 6)
        before = cache.k.clone()
        be.kv_append(cache, k, k, i32(lens), counts=None if counts is None else i32(counts), index=None if index is None else i32(index))
        with pytest.raises(Lq4Error):
            be.check_device_status()
        be.check_device_status()                                                # cleared
        if bad_page:
            assert torch.equal(cache.k, before)


def test_append_python_refusals(be):
    cache = make_cache(2, 2, 4, 2, 16)
    k = on_gpu(normal(24, 2, 3, 2, 16), BF16)
    lens = torch.zeros(2, dtype=torch.int32).cuda()
    for bad in (dict(k=k[:1], v=k[:1]), dict(k=k[..., :8], v=k[..., :8]), dict(v=k.float()), dict(kv_lens=lens.long()), dict(kv_lens=lens.cpu()),
                dict(counts=lens[:1]), dict(index=lens), dict(k=k.cpu(), v=k.cpu())):
        with pytest.raises((ValueError, TypeError)):
            a = dict(k=k, v=k, kv_lens=lens)
            a.update(bad)
            be.kv_append(cache, a.pop("k"), a.pop("v"), a.pop("kv_lens"), **a)
