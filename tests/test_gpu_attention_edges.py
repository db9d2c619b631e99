"""The attention half of a step at the edges of what its calls allow, on the GPU."""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    from lattice_b200 import CudaQ4Backend
    b = CudaQ4Backend(0)
    yield b
    b.close()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


def dense_cache(batch, max_pages, page, heads, dim, seed=1):
    """A cache of known contents whose pages lie in order."""
    from lattice_b200 import KvCache
    shape = (batch * max_pages, page, heads, dim)
    k, v = (normal(seed + i, *shape).to(BF16).cuda() for i in range(2))
    return KvCache(k, v, torch.arange(batch * max_pages, dtype=torch.int32).view(batch, max_pages).cuda())


# ---- cache append --------------------------------------------------------------------------------------------------

def append_by_c(be, cache, rows, kv_lens, new_lens, counts=None):
    """lq4_kv_append as a C caller makes it, without rows to read."""
    from lattice_b200 import _lib
    args = _lib.KvAppendArgs(C.pointer(cache.desc), None, None, _lib.DTYPE_BF16, rows, 0, 0, 0, kv_lens.data_ptr(),
                             None if counts is None else counts.data_ptr(), None, None if new_lens is None else new_lens.data_ptr())
    return _lib.lib().lq4_kv_append(be._ctx, C.byref(args), torch.cuda.current_stream().cuda_stream)


def test_append_of_no_rows_writes_the_lengths(be):
    cache = dense_cache(4, 2, 8, 1, 16)
    lens, new = i32([5, 0, -3, 16]), i32([99, 99, 99, 99])
    assert append_by_c(be, cache, 0, lens, new) == 0
    assert new.tolist() == [5, 0, -3, 16]
    assert append_by_c(be, cache, 0, lens, None) == 0
    empty = torch.empty(4, 0, 1, 16, dtype=BF16).cuda()
    assert be.kv_append(cache, empty, empty, lens).tolist() == [5, 0, -3, 16]
    assert be.kv_append(cache, empty, empty, lens, new_lens=lens).tolist() == [5, 0, -3, 16]
    be.check_device_status()


@pytest.mark.parametrize("lens, counts, rows, want", [
    ([5], [-1], 3, [5]),                     # a negative count
    ([17], [0], 3, [16]),                    # a length above the capacity, nothing to add
    ([17], None, 0, [16]),                   # the same without any rows
    ([5], [1], 0, [5]),                      # a count above the rows there are
])
def test_append_reports_every_value_out_of_range(be, lens, counts, rows, want):
    from lattice_b200 import Lq4Error
    cache = dense_cache(1, 2, 8, 1, 16)
    before = cache.k.clone()
    x = normal(3, 1, rows, 1, 16).to(BF16).cuda()
    assert be.kv_append(cache, x, x, i32(lens), counts=None if counts is None else i32(counts)).tolist() == want
    with pytest.raises(Lq4Error):
        be.check_device_status()
    assert torch.equal(cache.k, before)


def test_append_reports_nothing_of_sequences_to_leave_alone(be):
    cache = dense_cache(2, 2, 8, 1, 16)
    x = normal(4, 2, 3, 1, 16).to(BF16).cuda()
    assert be.kv_append(cache, x, x, i32([-1, 16]), counts=i32([9, 0]), index=i32([[7, 7, 7], [-1, -1, -1]])).tolist() == [-1, 16]
    be.check_device_status()


# ---- attention -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("length", [50, 5000])
@pytest.mark.parametrize("hq, d", [(2, 64), (10, 64), (32, 64), (2, 128), (9, 128), (80, 128), (3, 256), (12, 256), (3, 192), (12, 192)])
def test_attention_over_a_cache_with_infinities(be, hq, d, length, dtype):
    """The weights of a softmax are positive: an infinity in a cached V row makes its column infinite for every row that sees
    it, two of different signs or a NaN make it NaN, and no other column changes, however light the key is."""
    b, t = 2, 4
    light, lens = 37, [length, length // 2]
    cache = dense_cache(b, -(-length // 16) + 1, 16, 1, d, seed=30)
    q = normal(31, b, t, hq, d).abs().to(dtype).cuda()
    k, v = normal(32, b, t, 1, d).to(BF16).cuda(), normal(33, b, t, 1, d).to(BF16).cuda()
    par = i32([[-1, 0, 0, 1]] * b)
    rows = lambda x: x.view(b, -1, 1, d)  # noqa: E731
    rows(cache.k)[:, light] = -30.0                                          # its weight underflows: below e^-100 of the others'
    clean = be.tree_attention(q, k, v, cache, i32(lens), parents=par).cpu()
    inf, nan = math.inf, math.nan
    c = rows(cache.v)
    c[0, 3, 0, 0], c[0, 11, 0, 1], c[0, 20, 0, 2] = inf, -inf, nan
    c[0, 5, 0, 3], c[0, 45, 0, 3] = inf, -inf
    c[0, light, 0, d - 1] = inf
    c[0, lens[0] - 1, 0, 9], c[0, light, 0, 9] = -inf, -inf
    c[0, 3, 0, 10] = inf
    v[0, 2, 0, 10] = -inf                                                    # node 2 sees both
    c[0, lens[0]:] = nan                                                     # nobody sees these
    got = be.tree_attention(q, k, v, cache, i32(lens), parents=par).cpu()
    want = clean.clone()
    for col, x in ((0, inf), (1, -inf), (2, nan), (3, nan), (d - 1, inf), (9, -inf), (10, inf)):
        want[0, :, :, col] = x
    want[0, 2, :, 10] = nan
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    be.check_device_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq, d", [(2, 64), (10, 64), (80, 64), (2, 128), (9, 128), (80, 128), (3, 256), (12, 256), (12, 192)])
def test_attention_over_many_caches_with_infinities(be, hq, d, dtype):
    """The same where a CTA has whole sequences, not parts of them; and a row whose weights are NaN stays NaN everywhere."""
    b, t, length = 500, 2, 100
    cache = dense_cache(b, 7, 16, 1, d, seed=40)
    q = normal(41, b, t, hq, d).to(dtype).cuda()
    k, v = normal(42, b, t, 1, d).to(BF16).cuda(), normal(43, b, t, 1, d).to(BF16).cuda()
    q[7::50, 1, 0, 5] = math.nan
    lens = i32([length - i % 3 for i in range(b)])
    clean = be.tree_attention(q, k, v, cache, lens).cpu()
    c = cache.v.view(b, -1, 1, d)
    c[::2, 31, 0, 3], c[::2, 64, 0, 4] = math.inf, -math.inf
    c[::3, 90, 0, 5], c[::3, 2, 0, 5] = math.inf, -math.inf
    got = be.tree_attention(q, k, v, cache, lens).cpu()
    want = clean.clone()
    want[::2, ..., 3], want[::2, ..., 4], want[::3, ..., 5] = math.inf, -math.inf, math.nan
    want[7::50, 1, 0] = math.nan
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    bits = got.view(torch.int16 if dtype == BF16 else torch.int32)
    assert not bool(((bits < 0) & got.isnan()).any())                        # no mark is left


@pytest.mark.parametrize("hq, d, keys", [(4, 128, 1 << 19), (40, 128, 1 << 19), (80, 128, 1 << 18), (200, 64, 1 << 18), (4, 256, 1 << 19), (24, 256, 1 << 19), (24, 192, 100032)])
def test_attention_over_long_pieces_has_no_bias(be, hq, d, keys):
    """One CTA sums thousands of tiles of values of one sign: a sum that cuts off its last bits is low by more the longer it
    gets.  148 sequences share one set of pages, so that each CTA has whole items; the columns' means are spread over two
    binades, so that the roundings of the results do not add up."""
    from lattice_b200 import KvCache
    b, page = 148, 64
    g = torch.Generator(device="cuda").manual_seed(50)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    mean = 0.5 + 1.5 * (torch.arange(d, device="cuda") + 0.5) / d
    k = draw(keys // page, page, 1, d).to(BF16)
    v = (mean * (1 + 0.3 * draw(keys // page, page, 1, d))).to(BF16)
    table = torch.arange(keys // page, dtype=torch.int32, device="cuda").expand(b, -1).contiguous()
    q, kn, vn = draw(b, 1, hq, d).to(BF16), draw(b, 1, 1, d).to(BF16), mean.to(BF16).expand(b, 1, 1, d)
    lens = torch.full((b,), keys, dtype=torch.int32, device="cuda")
    got = be.tree_attention(q, kn, vn, KvCache(k, v, table), lens)
    be.check_device_status()
    off = []
    for i in (0, 77, 147):
        kk, vv = torch.cat([k.view(keys, d), kn[i, 0]]).double(), torch.cat([v.view(keys, d), vn[i, 0]]).double()
        ref = torch.softmax(q[i, 0].double() @ kk.T * d ** -0.5, -1) @ vv
        err = (got[i, 0].double() - ref) / ref
        # half a step of the result, and half a step of each weight (their sum's errors average out: 0.3 of it at most)
        assert float(err.abs().max()) <= 2.0 ** -8 + 0.3 * 2.0 ** -8
        off.append(float(err.mean()))
    # The results' roundings: uniform within half a step, an rms of 2^-8 / 3^0.5, one of its own per column and five standard
    # deviations of their mean.  A cut-off of half a last bit (2^-24) on average at each of the MMAs that one sum goes through:
    # at most four a tile for 512 tiles, which are then summed up in f32.
    assert abs(sum(off)) / 3 <= 5 * 2.0 ** -8 / (3 * d) ** 0.5 + 4 * 512 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq, d", [(4, 64), (9, 128), (24, 128), (40, 128), (200, 128), (140, 64), (3, 256), (24, 256), (12, 192)])
def test_attention_of_items_in_several_pieces(be, hq, d, dtype):
    """Sequences of 500 to 1600 tiles, whose pieces end at 512 tiles, at the items' and at the CTAs' borders."""
    from lattice_b200 import KvCache
    b, page, most = 151, 48, 102400
    g = torch.Generator(device="cuda").manual_seed(60)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    k, v = draw(-(-most // page), page, 1, d).to(BF16), draw(-(-most // page), page, 1, d).to(BF16)
    table = torch.arange(k.shape[0], dtype=torch.int32, device="cuda").expand(b, -1).contiguous()
    q, kn, vn = draw(b, 1, hq, d).to(dtype), draw(b, 1, 1, d).to(BF16), draw(b, 1, 1, d).to(BF16)
    lens = [32000 + (i * 7919) % 70000 for i in range(b)]
    lens[0], lens[1], lens[2], lens[3] = 511 * 64, 511 * 64 + 1, 512 * 64 + 1, 0
    q[1] *= 30.0 / d ** 0.5                                                  # sharp weights too: the maximum moves late
    got = be.tree_attention(q, kn, vn, KvCache(k, v, table), i32(lens))
    assert torch.equal(got, be.tree_attention(q, kn, vn, KvCache(k, v, table), i32(lens)))
    be.check_device_status()
    for i in (0, 1, 2, 3, 50, 77, 149, 150):
        n = lens[i]
        kk, vv = torch.cat([k.view(-1, d)[:n], kn[i, 0]]).double(), torch.cat([v.view(-1, d)[:n], vn[i, 0]]).double()
        x = q[i, 0].double()
        w = torch.softmax(x @ kk.T * d ** -0.5, -1)
        ref, mag, size = w @ vv, w @ vv.abs(), (x.norm(dim=-1) * kk.norm(dim=-1).amax() * d ** -0.5)[:, None]
        # products are exact, about 16 roundings of 2^-23 of at most |q| |k| scale lie in a score, two more in the exponent and
        # 2^-22 in exp2, each counts twice; four cut-offs of 2^-23 a tile for 512 tiles with bf16 activations, else one a
        # tile, and the joins; half a step for bf16 weights, and of the result
        e = 2 * (16 * 2.0 ** -23 * size + 2.0 ** -21) + (4 * 512 if dtype == BF16 else n / 64 + 200) * 2.0 ** -23
        half = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
        tol = mag * (e + (half if dtype == BF16 else 0.0)) + half * ref.abs() * 1.01
        err = (got[i, 0].double() - ref).abs()
        assert bool((err <= tol).all()), (i, float((err / tol).max()))


# ---- verification of drafted tokens --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("batch, vocab", [(3, 40), (3, 300), (80, 20011), (3, 70000)])      # (the last: row statistics first)
def test_verify_at_an_infinite_temperature(be, batch, vocab, sampled, dtype):
    """All logits above -inf weigh the same: one of n is accepted below 1 / n, and the last token is the one that the uniform
    points at.  The logits' size no longer counts, and the rows' padding has no mass."""
    g = torch.Generator().manual_seed(5)
    target = (30 * torch.randn(batch, 3, vocab, generator=g)).to(dtype)
    target[:, :, ::4] = -math.inf                                            # a quarter (rounded up) is masked out
    n = vocab - (vocab + 3) // 4
    draft = torch.randn(batch, 3, vocab, generator=g).to(dtype) if sampled else None      # all of them: 1 / vocab each
    tokens = torch.full((batch, 3), 1, dtype=torch.int32)
    u = torch.full((batch, 3), 0.5)
    u[:, 0] = (n // 2 + 0.5) / n                                             # in the middle of an entry
    u[:, 1] = 0.999 if sampled else 0.5 / n                                  # accepted: u / vocab < 1 / n, or u < 1 / n
    u[::2, 2] = 0.5 if sampled else 1.5 / n
    tokens[:, 2] = 4                                                         # masked: refused
    tau = torch.full((batch,), math.inf)
    path, count, token = be.verify_draft(target.cuda(), tokens.cuda(), u.cuda(), draft_logits=None if draft is None else draft.cuda(), temperature=tau.cuda())
    assert path.tolist() == [[0, 1, -1]] * batch and count.tolist() == [2] * batch
    # behind the refusal: max(p - q, 0) is 1/n - 1/vocab on the unmasked ones, and without a draft token 4 had no mass either
    live = [j for j in range(vocab) if j % 4]
    assert token.tolist() == [live[n // 2]] * batch
    be.check_device_status()


# ---- streams, threads and graphs -----------------------------------------------------------------------------------

def attention_job(seed, nodes, hq, dtype=BF16, batch=2, length=3000):
    """A call that needs partials of its own, and what it gives when nothing else runs."""
    cache = dense_cache(batch, -(-length // 32) + 1, 32, 2, 128, seed=seed)
    q = normal(seed + 5, batch, nodes, hq, 128).to(dtype).cuda()
    k, v = normal(seed + 6, batch, nodes, 2, 128).to(BF16).cuda(), normal(seed + 7, batch, nodes, 2, 128).to(BF16).cuda()
    lens = i32([length - 7 * i for i in range(batch)])
    return lambda be, out=None: be.tree_attention(q, k, v, cache, lens, out=out)


def verify_job(seed, vocab=70000):
    """A chain whose row statistics come first."""
    g = torch.Generator().manual_seed(seed)
    target = (2 * torch.randn(2, 5, vocab, generator=g)).cuda()
    draft = target + 0.3 * torch.randn(2, 5, vocab, generator=g).cuda()
    tokens, u = draft.argmax(-1).roll(1, 1).to(torch.int32), torch.rand(2, 5, generator=g).cuda()
    return lambda be: torch.cat([x.flatten() for x in be.verify_draft(target, tokens, u, draft_logits=draft)])


JOBS = [lambda s=s, shape=shape: attention_job(10 * s, *shape) for s, shape in enumerate([(1, 8), (16, 8), (5, 6, F32), (64, 8), (1, 24, F32)])] + \
       [lambda s=s: verify_job(100 + s) for s in range(3)]


@pytest.mark.parametrize("n_streams", [2, 8])
def test_one_backend_on_several_streams(n_streams):
    """Calls that run side by side do not disturb one another's workspaces, however many streams there are."""
    from lattice_b200 import CudaQ4Backend
    be = CudaQ4Backend(0)
    jobs = [make() for make in JOBS][:n_streams] if n_streams > 2 else [JOBS[0](), JOBS[1]()]
    want = [job(be).clone() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for turn in range(30):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[(i + turn // 10) % len(streams)]):
                got[i].append(job(be))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)
    be.check_device_status()
    be.close()


def test_one_backend_on_several_threads():
    """Each thread has its own stream and its own packed arguments."""
    import threading
    from lattice_b200 import CudaQ4Backend
    be = CudaQ4Backend(0)
    jobs = [make() for make in JOBS]
    want = [job(be).clone() for job in jobs]
    torch.cuda.synchronize()
    wrong, failed = [], []

    def work(job, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [job(be) for _ in range(60)]
                torch.cuda.current_stream().synchronize()
                wrong.extend(o for o in outs if not torch.equal(o, w))
        except Exception as e:                                               # (an exception in a thread does not end the test)
            failed.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and not wrong
    be.check_device_status()
    be.close()


def test_two_graphs_of_one_backend_side_by_side():
    """Graphs captured from one backend, without a plain call before, replay on two streams at once beside eager calls."""
    from lattice_b200 import CudaQ4Backend
    be, other = CudaQ4Backend(0), CudaQ4Backend(0)
    jobs = [make() for make in JOBS]
    want = [job(other).clone() for job in jobs]
    graphs, outs = [], []
    for job in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([job(be), job(be)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = [job(be) for job in jobs]
    torch.cuda.synchronize()
    for w, pair, e in zip(want, outs, eager):
        assert torch.equal(w, pair[0]) and torch.equal(w, pair[1]) and torch.equal(w, e)
    be.check_device_status()
    be.close()
    other.close()


@pytest.mark.parametrize("known", [True, False])
def test_an_eager_call_beside_a_capture(known):
    """While one stream captures, another one may call, also for the first time, and take or grow a workspace."""
    from lattice_b200 import CudaQ4Backend
    be, other = CudaQ4Backend(0), CudaQ4Backend(0)
    cache, lens = dense_cache(2, 60, 32, 2, 128, seed=70), i32([1800, 1700])
    q, k, v = (normal(71 + i, 2, 3, h, 128).to(BF16).cuda() for i, h in enumerate((16, 2, 2)))
    want = other.tree_attention(q, k, v, cache, lens)
    side, outs = torch.cuda.Stream(), [torch.zeros_like(q) for _ in range(2)]
    torch.cuda.synchronize()
    if known:
        with torch.cuda.stream(side):
            be.tree_attention(q, k, v, cache, lens, out=outs[1])
        torch.cuda.synchronize()
        outs[1].zero_()
        torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.tree_attention(q, k, v, cache, lens, out=outs[0])
        with torch.cuda.stream(side):
            be.tree_attention(q, k, v, cache, lens, out=outs[1])
    side.synchronize()
    assert torch.equal(outs[1], want)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    be.check_device_status()
    be.close()
    other.close()


def test_a_graph_that_grows_inside_its_capture():
    """A wider call later in a capture takes a larger workspace; the calls before it keep theirs."""
    from lattice_b200 import CudaQ4Backend
    be, other = CudaQ4Backend(0), CudaQ4Backend(0)
    small, large = JOBS[0](), JOBS[3]()
    want = small(other).clone(), large(other).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [small(be), large(be), small(be)]
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(outs[2], want[0])
    be.close()
    other.close()


def test_workspaces_of_dropped_graphs_are_taken_over():
    import gc
    from lattice_b200 import CudaQ4Backend
    be = CudaQ4Backend(0)
    job = JOBS[3]()
    want = job(be).clone()
    room = []
    for _ in range(24):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = job(be)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del g, out
        gc.collect()
        room.append(torch.cuda.mem_get_info()[0])
    assert room[3] - room[-1] < 64 << 20                                     # (a workspace of this call takes 39 MB)
    be.close()


def test_no_growth():
    """Without growth: attention takes what the first stream has or refuses, verification does without statistics."""
    from lattice_b200 import CudaQ4Backend, Lq4Error, _lib
    be = CudaQ4Backend(0)
    small, large, verify = JOBS[0](), JOBS[3](), JOBS[5]()
    with_stats = verify(CudaQ4Backend(0))
    want = small(be).clone()
    be.set_option(_lib.OPT_ALLOW_GROW, 0)
    with pytest.raises(Lq4Error, match="growth"):
        large(be)
    before = be.launch_count
    assert torch.equal(verify(be), with_stats) and be.launch_count == before + 1
    assert torch.equal(small(be), want)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert torch.equal(small(be), want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = small(be)
    g.replay()
    assert torch.equal(out, want)
    fresh = CudaQ4Backend(0)
    fresh.set_option(_lib.OPT_ALLOW_GROW, 0)
    with pytest.raises(Lq4Error, match="growth"):
        small(fresh)
    be.close()
    fresh.close()
