"""Rotary positions, cache append, tree attention and draft verification on the GPU, against plain 64-bit implementations."""
import itertools
import math
from fractions import Fraction

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
    (33, 24, 256, 64, BF16, BF16), (2, 1, 1024, 1024, F32, F32), (1000, 1, 6, 4, F32, BF16), (5, 3, 72, 16, BF16, BF16), (9, 3, 602, 300, F32, BF16), (40, 7, 1022, 10, BF16, F32),
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


# ---- tree attention ------------------------------------------------------------------------------------------------

def random_tree(seed, batch, nodes, width):
    """[batch, nodes] parents: each node hangs on one of the `width` nodes before it, or on the cached sequence."""
    at = torch.arange(nodes)
    back = (torch.rand(batch, nodes, generator=rng(seed)) * (at + 1).clamp(max=width)).long()
    return (at - 1 - back).clamp(min=-1).to(torch.int32)


def paths_of(parents, n):
    """Per node the nodes it sees: itself and its ancestors."""
    out = []
    for t in range(n):
        at, path = t, []
        while at >= 0:
            path.append(at)
            at = int(parents[at]) if parents is not None else at - 1
        out.append(path)
    return out


def attend_ref(q, k, v, cache_k, cache_v, table, lens, parents, counts, scale):
    """64-bit attention by the definition, one sequence after the other; also the weighted magnitudes of v and the
    size of the scores, for the tolerances.  Rows of dead nodes are NaN."""
    batch, nodes, heads, dim = q.shape
    hk, page = k.shape[2], cache_k.shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    mag, size = torch.zeros_like(out), torch.zeros(batch, nodes, heads, 1, dtype=torch.float64)
    for b in range(batch):
        n = lens[b]
        live = nodes if counts is None else counts[b]
        if n < 0:
            continue
        at = [(int(table[b, s // page]), s % page) for s in range(n)]
        idx = torch.tensor(at, dtype=torch.long).view(-1, 2)
        kk = torch.cat([cache_k[idx[:, 0], idx[:, 1]], k[b]]).double().repeat_interleave(heads // hk, 1)
        vv = torch.cat([cache_v[idx[:, 0], idx[:, 1]], v[b]]).double().repeat_interleave(heads // hk, 1)
        for t, path in enumerate(paths_of(parents[b] if parents is not None else None, live)):
            keys = torch.tensor(list(range(n)) + [n + j for j in sorted(path)])
            s = torch.einsum("hd,nhd->hn", q[b, t].double(), kk[keys]) * scale
            w = torch.softmax(s, -1)
            out[b, t] = torch.einsum("hn,nhd->hd", w, vv[keys])
            mag[b, t] = torch.einsum("hn,nhd->hd", w, vv[keys].abs())
            size[b, t, :, 0] = (q[b, t].double().norm(dim=-1) * kk[keys].norm(dim=-1).amax(0)) * abs(scale)
    return out, mag, size


def assert_attention(got, ref, mag, size, keys):
    """Scores: products are exact, about 16 roundings of 2^-23 of at most |q| |k| scale lie in a sum, two more in the
    exponent and 2^-22 in exp2; each error counts twice (numerator and sum).  bf16 activations: probabilities and result
    are rounded by half a step of 2^-8.  The running sums round once a tile of 64 keys, and at the joins."""
    e = 2 * (16 * 2.0 ** -23 * size + 2.0 ** -21) + (keys / 64 + 200) * 2.0 ** -23
    if got.dtype == BF16:
        e = e + 2.0 ** -8
    tol = mag * e + HALF_STEP[got.dtype] * ref.abs() * 1.01 + 1e-30
    err = (got.double().cpu() - ref).abs()
    live = ~ref.isnan()
    assert bool((err <= tol)[live].all()), float((err / tol)[live].max())


def attend_case(be, seed, batch, nodes, hq, hk, dim, page, lens, dtype, width=2, counts=None, order="dense", scale=None, poison=True, chain=False):
    """Random inputs with NaN in every cache slot behind a sequence's length, run and checked."""
    most = max(max(lens), 0)
    cache = make_cache(batch, -(-max(most, 1) // page) + 1, page, hk, dim, seed=seed, order=order)
    if poison:
        keep = torch.zeros(cache.k.shape[:2], dtype=torch.bool)
        table = cache.page_table.cpu().long()
        for b, n in enumerate(lens):
            s = torch.arange(max(n, 0))
            keep[table[b, s // page], s % page] = True
        for x in (cache.k, cache.v):
            x.masked_fill_(~keep[:, :, None, None].cuda(), math.nan)
    q = (2 * normal(seed + 5, batch, nodes, hq, dim)).to(dtype)
    k, v = (normal(seed + 6 + i, batch, nodes, hk, dim).to(BF16) for i in range(2))
    parents = None if chain or nodes == 1 else random_tree(seed + 8, batch, nodes, width)
    i32 = lambda x: None if x is None else torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    out = torch.full(q.shape, 7.0, dtype=dtype).cuda()
    got = be.tree_attention(q.cuda(), k.cuda(), v.cuda(), cache, i32(lens), parents=i32(parents), node_counts=i32(counts), scale=scale, out=out)
    ref = attend_ref(q, k, v, cache.k.cpu(), cache.v.cpu(), cache.page_table.cpu(), lens, parents, counts, dim ** -0.5 if scale is None else scale)
    assert_attention(got, *ref, most + nodes)
    dead = ref[0].isnan()
    assert bool((got.cpu()[dead] == 7.0).all())                                  # rows of nobody stay as they were
    be.check_device_status()
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("length", [0, 1, 5, 63, 64, 65, 127, 1000])
def test_attention_lengths_of_one_token(be, dtype, length):
    attend_case(be, 100 + length, 2, 1, 10, 2, 128, 16, [length, max(length - 1, 0)], dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim, hq, hk", [(8, 1, 1), (64, 4, 4), (72, 6, 2), (80, 16, 1), (128, 5, 1), (192, 8, 2), (256, 12, 2), (256, 3, 1)])
@pytest.mark.parametrize("nodes", [1, 5, 16, 64])
def test_attention_shapes(be, dtype, dim, hq, hk, nodes):
    """All bands of rows (16, 32, 64, several tiles) and all padded head sizes."""
    attend_case(be, 7 * dim + nodes, 2, nodes, hq, hk, dim, 24, [150, 33], dtype, width=4)


@pytest.mark.parametrize("page", [1, 5, 7, 64, 100])
@pytest.mark.parametrize("order", ["dense", "heads"])
def test_attention_pages_that_end_inside_a_tile(be, page, order):
    attend_case(be, page, 3, 3, 4, 2, 64, page, [131, 64, 0], BF16, order=order)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_ragged_batch_with_dead_rows(be, dtype):
    lens = [17, -1, 400, 0, 64, 1, -5, 900]
    counts = [6, 6, 1, 3, 0, 6, 2, 5]
    attend_case(be, 40, 8, 6, 6, 3, 64, 16, lens, dtype, counts=counts, width=3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nodes, hq", [(2, 2), (5, 8)])
def test_attention_large_ragged_batch(be, nodes, hq, dtype):
    lens = [(37 * i) % 300 - 1 for i in range(300)]
    attend_case(be, 41, 300, nodes, hq, 1, 64, 32, lens, dtype, poison=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_long_sequences_are_split(be, dtype):
    """One item over every CTA, with a border inside a page; chains and trees."""
    attend_case(be, 42, 1, 4, 4, 1, 128, 48, [20011], dtype, width=2)
    attend_case(be, 43, 2, 7, 5, 1, 256, 16, [3000, 9000], dtype, chain=True)
    attend_case(be, 45, 1, 16, 8, 1, 128, 48, [20011], dtype, width=3)
    attend_case(be, 46, 2, 64, 8, 2, 64, 5, [5000, 777], dtype, width=5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 128, 129, 256, 257])
def test_attention_rows_at_the_kernels_borders(be, dtype, rows):
    """Rows per kv head where another kernel or another number of row tiles takes over: one node of `rows` query heads."""
    attend_case(be, rows, 2, 1, rows, 1, 72, 16, [70, 129], dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nodes, hq, d", [(3, 4, 64), (5, 24, 64), (64, 6, 128), (9, 8, 256)])
def test_attention_unaligned_rows(be, nodes, hq, d, dtype):
    """q and out with odd strides and offsets, which no vector access fits."""
    b, hk = 2, 2
    cache = make_cache(b, 8, 16, hk, d, seed=55)
    q = (2 * normal(56, b, nodes, hq, d)).to(dtype)
    k, v = normal(57, b, nodes, hk, d).to(BF16), normal(58, b, nodes, hk, d).to(BF16)
    shape, stride = (b, nodes, hq, d), (nodes * (hq * (d + 1) + 3) + 1, hq * (d + 1) + 3, d + 1, 1)
    room = torch.zeros(2, b * stride[0] + 8, dtype=dtype).cuda()
    qs, out = torch.as_strided(room[0], shape, stride, 1), torch.as_strided(room[1], shape, stride, room.shape[1] + 3)
    qs.copy_(q)
    lens, par = [100, 65], random_tree(59, b, nodes, 2)
    dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = be.tree_attention(qs, k.cuda(), v.cuda(), cache, dev(lens), parents=dev(par), out=out)
    ref = attend_ref(q, k, v, cache.k.cpu(), cache.v.cpu(), cache.page_table.cpu(), lens, par, None, d ** -0.5)
    assert_attention(got, *ref, 164)
    room[1].as_strided(shape, stride, room.shape[1] + 3).zero_()
    assert not room[1].any()                                                     # nothing between the rows was written


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(be, scale):
    attend_case(be, 44, 2, 5, 4, 2, 64, 16, [100, 7], F32, scale=scale)


def test_attention_strided_rows_and_same_bits_again(be):
    """q, k and v as slices of one fused row, out as a slice; the same call gives the same bits."""
    b, t, hq, hk, d = 3, 4, 6, 2, 64
    fused = normal(50, b, t, hq + 2 * hk, d).to(BF16)
    g = fused.cuda()
    cache = make_cache(b, 8, 16, hk, d, seed=51)
    lens = [100, 3, 65]
    par = random_tree(52, b, t, 2)
    wide = torch.zeros(b, t, 2 * hq, d, dtype=BF16).cuda()
    q, k, v = g.split([hq, hk, hk], 2)
    dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    got = be.tree_attention(q, k, v, cache, dev(lens), parents=dev(par), out=wide[:, :, hq:])
    cq, ck, cv = fused.split([hq, hk, hk], 2)
    assert_attention(got, *attend_ref(cq, ck, cv, cache.k.cpu(), cache.v.cpu(), cache.page_table.cpu(), lens, par, None, d ** -0.5), 104)
    assert not wide[:, :, :hq].any()
    again = be.tree_attention(q, k, v, cache, dev(lens), parents=dev(par))
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq, d", [(2, 64), (32, 64), (12, 128), (80, 128), (8, 256)])
def test_attention_masked_nodes_hold_anything(be, hq, d, dtype):
    """Node 1 and node 2 are siblings; what node 2 holds reaches node 2 only."""
    b, t = 1, 4
    cache = make_cache(b, 4, 16, 1, d, seed=60)
    q = normal(61, b, t, hq, d).to(dtype)
    k, v = normal(62, b, t, 1, d).to(BF16), normal(63, b, t, 1, d).to(BF16)
    par = torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32)
    lens = torch.tensor([50], dtype=torch.int32).cuda()
    clean = be.tree_attention(q.cuda(), k.cuda(), v.cuda(), cache, lens, parents=par.cuda()).cpu()
    v2 = v.clone()
    v2[0, 2, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, math.inf])
    dirty = be.tree_attention(q.cuda(), k.cuda(), v2.cuda(), cache, lens, parents=par.cuda()).cpu()
    assert torch.equal(dirty[:, [0, 1, 3]], clean[:, [0, 1, 3]])
    for h in range(hq):
        assert dirty[0, 2, h, 0] == math.inf and dirty[0, 2, h, 1] == -math.inf and dirty[0, 2, h, 2].isnan()
    assert torch.equal(dirty[0, 2, :, 4:], clean[0, 2, :, 4:])
    for bad in (math.nan, math.inf, torch.finfo(BF16).min):
        k2, v3 = k.clone(), v2.clone()
        k2[0, 2] = bad
        v3[0, 2] = bad
        dirty = be.tree_attention(q.cuda(), k2.cuda(), v3.cuda(), cache, lens, parents=par.cuda()).cpu()
        assert torch.equal(dirty[:, [0, 1, 3]], clean[:, [0, 1, 3]])


@pytest.mark.parametrize("hq", [2, 16])
def test_attention_reports_bad_indexes(be, hq):
    from lattice_b200 import Lq4Error
    d = 64
    q, k = normal(70, 1, 3, hq, d).to(BF16).cuda(), normal(71, 1, 3, 1, d).to(BF16).cuda()
    dev = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    for what in ("page", "negative page", "length", "count", "parent", "parent of itself"):
        cache = make_cache(1, 4, 16, 1, d, seed=72)
        lens, par, counts = [40], [[-1, 0, 1]], None
        if what == "page":
            cache.page_table[0, 1] = cache.k.shape[0]
        if what == "negative page":
            cache.page_table[0, 1] = -7
        if what == "length":
            lens = [65]
        if what == "count":
            counts = dev([4])
        if what == "parent":
            par = [[-1, 2, 0]]
        if what == "parent of itself":
            par = [[0, 0, 1]]
        got = be.tree_attention(q, k, k, cache, dev(lens), parents=dev(par), node_counts=counts)
        with pytest.raises(Lq4Error):
            be.check_device_status()
        be.check_device_status()
        if "page" in what:                                                       # the keys of that page are not seen
            keep = [s for s in range(40) if s // 16 != 1]
            kk = cache.k.cpu()[cache.page_table.cpu()[0, [0, 2]].long()].reshape(-1, 1, d)
            kk = torch.cat([kk[:16], kk[16:24]])
            assert len(keep) == kk.shape[0]
            vv = cache.v.cpu()[cache.page_table.cpu()[0, [0, 2]].long()].reshape(-1, 1, d)
            vv = torch.cat([vv[:16], vv[16:24]])
            ref = attend_ref(q.cpu(), k.cpu(), k.cpu(), kk[None], vv[None], torch.zeros(1, 1, dtype=torch.int32), [24], torch.tensor(par), None, d ** -0.5)
            assert_attention(got, *ref, 64)


@pytest.mark.parametrize("hq", [4, 24])
def test_attention_in_a_captured_graph(be, hq):
    """A graph replays with other lengths, pages and values; the launch does not depend on them."""
    b, t, d = 2, 3, 64
    cache = make_cache(b, 40, 16, 2, d, seed=80)
    q, k, v = normal(81, b, t, hq, d).to(BF16).cuda(), normal(82, b, t, 2, d).to(BF16).cuda(), normal(83, b, t, 2, d).to(BF16).cuda()
    lens, par = torch.tensor([5, 600], dtype=torch.int32).cuda(), random_tree(84, b, t, 2).cuda()
    out = torch.empty(b, t, hq, d, dtype=BF16, device="cuda")
    call = lambda: be.tree_attention(q, k, v, cache, lens, parents=par, out=out)  # noqa: E731
    call()                                                                       # the workspace grows outside the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for new in ([5, 600], [639, 0], [64, -1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(normal(85 + new[0], b, t, hq, d).to(BF16))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        ref = attend_ref(q.cpu(), k.cpu(), v.cpu(), cache.k.cpu(), cache.v.cpu(), cache.page_table.cpu(), new, par.cpu(), None, d ** -0.5)
        assert_attention(out, *ref, 640)
        assert bool((out.cpu()[ref[0].isnan()] == 7.0).all())
    be.check_device_status()


def test_attention_graph_after_a_larger_call():
    """A call with more rows per kv head outgrows the workspace; a graph captured before it keeps its own."""
    from lattice_b200 import CudaQ4Backend
    be = CudaQ4Backend(0)
    cache = make_cache(1, 40, 64, 1, 128, seed=90)
    lens = torch.tensor([2500], dtype=torch.int32).cuda()
    make = lambda hq, n: [normal(91 + n, 1, n, h, 128).to(BF16).cuda() for h in (hq, 1, 1)]  # noqa: E731
    small, large = make(4, 1), make(4, 64)
    out = torch.empty_like(small[0])
    eager = be.tree_attention(*small, cache, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.tree_attention(*small, cache, lens, out=out)
    big = be.tree_attention(*large, cache, lens)
    out.fill_(7.0)
    g.replay()
    assert torch.equal(out, eager)
    assert torch.equal(be.tree_attention(*large, cache, lens), big)
    be.check_device_status()
    be.close()


def test_attention_python_refusals(be):
    cache = make_cache(2, 2, 16, 2, 64)
    q, k = normal(90, 2, 3, 4, 64).to(BF16).cuda(), normal(91, 2, 3, 2, 64).to(BF16).cuda()
    lens = torch.zeros(2, dtype=torch.int32).cuda()
    for bad in (dict(q=q[:1]), dict(q=q[:, :2]), dict(q=q.half()), dict(q=q.cpu()), dict(k=k.float(), v=k.float()), dict(k=k[:, :, :1], v=k[:, :, :1]),
                dict(parents=lens), dict(kv_lens=lens.long()), dict(out=q.float()), dict(node_counts=lens[:1])):
        a = dict(q=q, k=k, v=k, kv_lens=lens)
        a.update(bad)
        with pytest.raises((ValueError, TypeError)):
            be.tree_attention(a.pop("q"), a.pop("k"), a.pop("v"), cache, a.pop("kv_lens"), **a)


# ---- verification of drafted tokens --------------------------------------------------------------------------------

def distribution(logits, tau):
    """softmax(logits / tau) in 64 bits; NaN and -inf carry nothing, +inf takes all; None for a row without mass."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return None
    w = (x == m).astype(np.float64) if m == np.inf else np.exp((x - m) / tau)
    return w / w.sum()


def verify_ref(target, draft, tokens, parents, n, uniforms, tau):
    """One sequence by the definition: residual distributions as vectors, renormalised after every refusal."""
    nodes, vocab = target.shape
    if n <= 0:
        return [-1] * nodes, 0, -1
    path, cur = [0], 0
    while True:
        children = [c for c in range(cur + 1, n) if (parents[c] if parents is not None else c - 1) == cur]
        if tau < 1e-20:
            x = np.where(np.isnan(target[cur]), -np.inf, target[cur])
            best = int(np.argmax(x)) if x.max() > -np.inf else -1
            step = next((c for c in children if tokens[c] == best and best >= 0), None)
        else:
            p = distribution(target[cur], tau)
            q = distribution(draft[cur], tau) if draft is not None else None
            left, step = (p if p is not None else np.zeros(vocab)), None
            gone = set()
            for c in children:
                t = int(tokens[c])
                if not 0 <= t < vocab:
                    continue
                u = float(uniforms[c])
                if draft is not None:
                    qt = q[t] if q is not None else 0.0
                    if u * qt < left[t]:
                        step = c
                        break
                    left = np.maximum(left - q, 0) if q is not None else left
                    left = left / left.sum() if left.sum() > 0 else left
                else:
                    if t in gone:
                        continue
                    if u < left[t]:
                        step = c
                        break
                    gone.add(t)
                    left = left.copy()
                    left[t] = 0
                    left = left / left.sum() if left.sum() > 0 else left
        if step is None:
            break
        path.append(step)
        cur = step
    if tau < 1e-20:
        token = best
    elif p is None:
        token = -1
    else:
        left = left if left.sum() > 0 else p
        if vocab <= 1000:                                                        # sums without rounding: equal masses can meet a border exactly
            total = np.array(list(itertools.accumulate(Fraction(x) for x in left.tolist())))
            border = Fraction(float(uniforms[0])) * total[-1]
        else:
            total = np.cumsum(left)
            border = float(uniforms[0]) * total[-1]
        over = np.nonzero(total > border)[0]
        token = int(over[0]) if len(over) else int(np.nonzero(left)[0][-1])
    return path + [-1] * (nodes - len(path)), len(path), token


def check_verify(be, target, draft, tokens, parents, counts, uniforms, tau):
    gpu = lambda x: None if x is None else x.cuda()  # noqa: E731
    got = be.verify_draft(gpu(target), gpu(tokens), gpu(uniforms), draft_logits=gpu(draft), parents=gpu(parents), node_counts=gpu(counts), temperature=gpu(tau))
    path, count, token = (x.cpu().numpy() for x in got)
    for b in range(target.shape[0]):
        ref = verify_ref(target[b].float().numpy(), None if draft is None else draft[b].float().numpy(), tokens[b].numpy(),
                         None if parents is None else parents[b].numpy(), target.shape[1] if counts is None else int(counts[b]),
                         uniforms[b].numpy(), 1.0 if tau is None else float(tau[b]))
        assert path[b].tolist() == ref[0] and count[b] == ref[1] and token[b] == ref[2], (b, path[b].tolist(), int(count[b]), int(token[b]), ref)
    be.check_device_status()
    return path, count, token


def verify_inputs(seed, batch, nodes, vocab, dtype, sampled, width=3, spread=2.0):
    g = rng(seed)
    target = (spread * torch.randn(batch, nodes, vocab, generator=g)).to(dtype)
    draft = (target.float() + 0.7 * torch.randn(batch, nodes, vocab, generator=g)).to(dtype)
    at = torch.arange(nodes)
    parents = (at - 1 - (torch.rand(batch, nodes, generator=g) * at.clamp(max=width)).long()).clamp(min=-1).to(torch.int32)
    of_parent = torch.take_along_dim(draft.float(), parents.clamp(min=0).long()[..., None], 1)
    noise = -torch.log(-torch.log(torch.rand(batch, nodes, vocab, generator=g).clamp(1e-30, 1 - 1e-7)))
    tokens = (of_parent + noise).argmax(-1).to(torch.int32)
    return target, draft if sampled else None, tokens, parents, torch.rand(batch, nodes, generator=g)


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 256, 257, 4099, 50001])
def test_verify_vocabularies(be, vocab, dtype, sampled):
    target, draft, tokens, parents, u = verify_inputs(vocab, 9, 7, vocab, dtype, sampled)
    tau = torch.tensor([0.0, 1.0, 0.5, 2.0, 1e-3, 1e-30, 1.0, 0.7, 0.7])
    check_verify(be, target, draft, tokens, parents, None, u, tau)


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("nodes, width", [(1, 1), (2, 1), (5, 1), (17, 4), (64, 8), (64, 63)])
def test_verify_trees(be, nodes, width, sampled):
    """Chains, trees and a star; few distinct tokens, so that siblings repeat one another; dead nodes."""
    target, draft, tokens, parents, u = verify_inputs(200 + nodes + width, 60, nodes, 23, F32, sampled, width)
    counts = torch.randint(0, nodes + 1, (60,), generator=rng(3), dtype=torch.int32)
    counts[:30] = nodes
    path, count, _ = check_verify(be, target, draft, tokens, parents if width > 1 else None, counts, u, None)
    if nodes > 4:
        assert count.max() >= 3                                                  # the walk goes deep in some of them


def test_verify_large_batch_and_full_vocabulary(be):
    target, draft, tokens, parents, u = verify_inputs(4, 300, 4, 1000, BF16, True)
    check_verify(be, target, draft, tokens, parents, None, u, None)
    target, draft, tokens, parents, u = verify_inputs(5, 2, 6, 248320, F32, True)
    check_verify(be, target, draft, tokens, parents, None, u, torch.tensor([0.9, 0.0]))


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_rows_too_long_for_the_registers(be, dtype, sampled):
    """80 sequences leave one CTA for each, and its warps' shares of a row are read again instead of being kept."""
    target, draft, tokens, parents, u = verify_inputs(6, 80, 4, 20011, dtype, sampled)
    tau = torch.ones(80)
    tau[::7], tau[1::7] = 0.0, 0.6
    check_verify(be, target, draft, tokens, parents, None, u, tau)


@pytest.mark.parametrize("vocab", [300, 50001])
def test_verify_in_a_captured_graph(vocab):
    """A graph replays with other logits, tokens and uniforms, also after a call that needs a larger workspace."""
    from lattice_b200 import CudaQ4Backend
    be = CudaQ4Backend(0)
    shape = (3, 5, vocab, F32, True)
    states = [verify_inputs(seed, *shape) for seed in (12, 13, 14)]
    target, draft, tokens, parents, u = (x.cuda() for x in states[0])
    call = lambda: be.verify_draft(target, tokens, u, draft_logits=draft, parents=parents)  # noqa: E731
    call()                                                                       # the workspace grows outside the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    check_verify(be, *verify_inputs(15, 9, 7, 60000, F32, True)[:4], None, torch.rand(9, 7, generator=rng(16)), None)
    for new in states:
        for x, y in zip((target, draft, tokens, parents, u), new):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        eager = check_verify(be, *new[:4], None, new[4], None)
        for x, y in zip(out, eager):
            assert x.cpu().numpy().tolist() == y.tolist()
    be.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_strange_rows(be, dtype):
    """Masked, infinite, NaN and empty rows; uniforms at the borders; tokens and parents out of range."""
    inf, nan = math.inf, math.nan
    target = torch.zeros(12, 3, 300).to(dtype)
    draft = torch.zeros(12, 3, 300).to(dtype)
    tokens = torch.full((12, 3), 5, dtype=torch.int32)
    u = torch.full((12, 3), 0.25)
    parents = torch.tensor([[-1, 0, 1]] * 12, dtype=torch.int32)
    target[0] = -inf                                                             # no mass: nothing accepted, token -1
    target[1, :, :299] = -inf                                                    # one entry has it all
    target[2, :, 7] = inf
    target[3, :, 100:] = nan
    draft[4] = -inf                                                              # a draft without mass: 0 < p accepts
    target[5, :, 5] = -inf                                                       # the drafted token is masked out
    draft[6, :, 5] = inf
    tokens[7] = -3
    tokens[8] = 300
    parents[9] = torch.tensor([5, 1, 7])                                         # no children of node 0
    u[10] = 0.0                                                                  # accepts; the first entry with mass
    target[10, :, :9] = -inf
    target[10, :, 5] = 0.0
    u[11] = 1.0 - 2.0 ** -24                                                     # the last one
    draft[11, :, 5] = 3.0
    for d in (draft, None):
        check_verify(be, target, d, tokens, parents, None, u, None)
        check_verify(be, target, d, tokens, parents, None, u, torch.zeros(12))


def test_verify_strides_and_same_again(be):
    wide = (2 * torch.randn(3, 5, 2, 77, generator=rng(8))).cuda()
    target, draft = wide[:, :, 0, 3:70], wide[:, :, 1, 3:70]
    tokens = torch.randint(0, 67, (3, 5), generator=rng(9), dtype=torch.int32)
    u = torch.rand(3, 5, generator=rng(10))
    a = be.verify_draft(target, tokens.cuda(), u.cuda(), draft_logits=draft)
    b = be.verify_draft(target.contiguous(), tokens.cuda(), u.cuda(), draft_logits=draft.contiguous())
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    check_verify(be, target.cpu().contiguous(), draft.cpu().contiguous(), tokens, None, None, u, None)


@pytest.mark.parametrize("sampled", [True, False])
def test_verify_keeps_the_targets_distribution(be, sampled):
    """The first token that a verification emits is distributed as the target says, whatever was drafted."""
    n, vocab = 60000, 6
    g = rng(11)
    target, draft = torch.randn(3, vocab, generator=g), torch.randn(3, vocab, generator=g)
    q = torch.softmax(draft[0], -1)
    tokens = torch.multinomial(q, 3 * n, True, generator=g).view(n, 3).to(torch.int32)   # nodes 1 and 2: siblings
    parents = torch.tensor([[-1, 0, 0]] * n, dtype=torch.int32)
    u = torch.rand(n, 3, generator=g)
    path, count, token = be.verify_draft(target.expand(n, 3, vocab).cuda(), tokens.cuda(), u.cuda(), parents=parents.cuda(),
                                         draft_logits=draft.expand(n, 3, vocab).cuda() if sampled else None)
    path, count, token = path.cpu().long(), count.cpu(), token.cpu()
    first = torch.where(count > 1, torch.gather(tokens, 1, path[:, 1:2].clamp(min=0))[:, 0], token)
    seen = torch.bincount(first, minlength=vocab).double() / n
    p = torch.softmax(target[0].double(), -1)
    assert bool(((seen - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all())        # five standard deviations of a frequency
    assert 0 < int((count > 1).sum()) < n


def test_verify_refusals(be):
    target, draft, tokens, parents, u = (x.cuda() for x in verify_inputs(12, 2, 3, 50, F32, True))
    for bad in (dict(draft_logits=draft.bfloat16()), dict(draft_logits=draft[:1]), dict(tokens=tokens.long()), dict(uniforms=u.double()), dict(uniforms=u[:1]),
                dict(parents=parents[:, :2]), dict(temperature=u), dict(target_logits=target.half()), dict(target_logits=target.cpu())):
        a = dict(target_logits=target, tokens=tokens, uniforms=u)
        a.update(bad)
        with pytest.raises((ValueError, TypeError)):
            be.verify_draft(a.pop("target_logits"), a.pop("tokens"), a.pop("uniforms"), **a)


# ---- a speculative decode step, all of it --------------------------------------------------------------------------

def test_two_backends_on_two_streams(be):
    """Each backend has its own workspace: two attentions that run side by side do not disturb one another."""
    from lattice_b200 import CudaQ4Backend
    other = CudaQ4Backend(0)
    calls, want = [], []
    for i, (b_, nodes, hq, dtype) in enumerate([(be, 1, 8, BF16), (other, 16, 8, BF16)]):
        cache = make_cache(2, 100, 32, 2, 128, seed=95 + i)
        q = normal(96 + i, 2, nodes, hq, 128).to(dtype).cuda()
        k = normal(97 + i, 2, nodes, 2, 128).to(BF16).cuda()
        lens = torch.tensor([3000, 1234], dtype=torch.int32).cuda()
        calls.append((b_, q, k, cache, lens))
        want.append(b_.tree_attention(q, k, k, cache, lens).clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(20):
        for i, (b_, q, k, cache, lens) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(b_.tree_attention(q, k, k, cache, lens))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)
    be.check_device_status()
    other.check_device_status()
    other.close()


@pytest.mark.parametrize("types", [BF16, F32])
def test_speculative_step(be, types):
    """Projections, rotary positions, attention of the tree, o_proj, lm_head over all nodes, verification, append, and the
    next step over what was accepted: every stage against 64 bits on the inputs that the GPU had."""
    from lattice_b200 import Q4WeightBuf, RopeTable, synth
    import oracle
    b, t, hidden, hq, hk, d, vocab = 2, 6, 256, 4, 2, 64, 1000
    weights = []
    for i, (n, k) in enumerate([((hq + 2 * hk) * d, hidden), (hidden, hq * d), (vocab, hidden)]):
        w = synth.weights(2, n, k, i)
        weights.append(Q4WeightBuf.from_host_payload(oracle.quantize_f32_to_q4(w), n, k))
    w_qkv, w_o, w_head = weights
    table = RopeTable.from_config(d, "cuda", theta=1e6)
    cache = make_cache(b, 12, 16, hk, d, seed=300)
    lens = torch.tensor([33, 90], dtype=torch.int32).cuda()
    draft_of = (2 * torch.randn(b, t, vocab, generator=rng(301))).cuda()
    for step in range(3):
        par = random_tree(302 + step, b, t, 2)
        par[:, 1:] = par[:, 1:].clamp(min=0)                                     # node 0 is the last certain token
        depth = torch.tensor([[len(p) - 1 for p in paths_of(par[i], t)] for i in range(b)])
        x = (normal(310 + step, b * t, hidden) * 0.5).float().cuda()
        fused = be.linear(x, w_qkv).view(b * t, hq + 2 * hk, d)
        pos = (lens[:, None].cpu() + depth).to(torch.int32).view(-1)
        q, k, v = fused.split([hq, hk, hk], 1)
        q, = be.rope_rows([(q, 1)], pos.cuda(), table, out_dtype=types)
        k, v = be.rope_rows([(k, 1), (v, 0)], pos.cuda(), table, out_dtype=BF16)
        for y, part in ((q, fused[:, :hq]), (k, fused[:, hq:hq + hk])):
            assert_rope(y, *rope_ref(part.cpu(), pos, table.freq.cpu().numpy(), "half", 1.0, 1))
        q, k, v = q.view(b, t, hq, d), k.view(b, t, hk, d), v.view(b, t, hk, d)
        att = be.tree_attention(q, k, v, cache, lens, parents=par.cuda())
        ref = attend_ref(q.cpu(), k.cpu(), v.cpu(), cache.k.cpu(), cache.v.cpu(), cache.page_table.cpu(), lens.tolist(), par, None, d ** -0.5)
        assert_attention(att, *ref, 200)
        logits = be.linear(be.linear(att.view(b * t, hq * d), w_o), w_head).view(b, t, vocab)
        assert bool(logits.isfinite().all())
        draft = logits + 0.3 * draft_of
        of_parent = torch.take_along_dim(draft, par.clamp(min=0).long()[..., None].cuda(), 1)
        tokens = (of_parent + -torch.log(-torch.log(torch.rand(of_parent.shape, generator=rng(320 + step)).clamp(1e-30, 1 - 1e-7))).cuda()).argmax(-1).to(torch.int32)
        u = torch.rand(b, t, generator=rng(330 + step))
        path, count, token = check_verify(be, logits.cpu(), draft.cpu(), tokens.cpu(), par, None, u, None)
        path, count = torch.from_numpy(path).cuda(), torch.from_numpy(count).cuda()
        # the last accepted node, attended alone once its ancestors are in the cache
        before = lens.clone()
        lens = be.kv_append(cache, k, v, before, counts=count - 1, index=path)
        last = torch.stack([path[i, count[i] - 1] for i in range(b)]).long()
        pick = lambda y: y[torch.arange(b).cuda(), last][:, None].contiguous()  # noqa: E731
        alone = be.tree_attention(pick(q), pick(k), pick(v), cache, lens)
        ref = [r[torch.arange(b), last.cpu()][:, None] for r in ref]
        assert_attention(alone, *ref, 200)
        lens = be.kv_append(cache, pick(k), pick(v), lens)
        assert (lens - before).tolist() == count.tolist()
    be.check_device_status()
    for w in weights:
        w.free()
