"""Edges of the paged 8-bit KV cache operators (rusty_engine_b200.kv) on the GPU, against
tests/kv_ref.py, with the tolerances of tests/test_kv.py unless a test derives its own."""
import numpy as np
import pytest
import torch

import kv_ref as R
from test_kv import REL, cache_of, ints, kv, rel, run_attend, slots_of  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- a dominant key -----------------------------------------------------------------------------
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("at", [0, 700])
@pytest.mark.parametrize("lens,new,nq,nkv,d", [
    ([1500], [1], 8, 2, 128), ([1500, 1300], [1, 3], 16, 2, 64), ([1400], [2], 4, 1, 256),
    ([1550], [200], 32, 8, 128), ([1550], [200], 32, 8, 64)])
def test_attend_beside_a_dominant_key(kv, code, dtype, at, lens, new, nq, nkv, d):
    """A key that takes nearly all of every row's weight while its value is 0: the output is what
    the other keys, 14 (f32) or 17 nats below, add up to.  f32: the deepest weight is 2^-22 of the
    row's largest; carried as 2^15 times itself in two fp16 it is off by at most 2^-25 / 2^-7, beside
    the 20 * 2^-22 of the scores: 1e-5 holds.  16 bits: weights of 2^-24.5 of the largest, carried
    as 2^7 times themselves, are rounded by at most 2^-25 each, the roundings of 1300 keys being
    independent: 2^-7.5 / sqrt(3 * 1300) = 1e-4 of the sum; 2^-11 is five times that."""
    depth, bs, g = (14.0 if dtype == "f32" else 17.0), 64, torch.Generator().manual_seed(d + at)
    _, _, table = slots_of(lens, [0] * len(lens), bs, blocks := sum(-(-n // bs) for n in lens))
    u = torch.randint(0, 2, (nkv, d), generator=g) * 2.0 - 1.0
    k = torch.randint(-20, 21, (blocks, nkv, bs, d), generator=g).float()
    v = (64 + 25 * torch.randn((blocks, nkv, bs, d), generator=g)).round().clamp(-127, 127)
    for row in table:
        k[row[at // bs], :, at % bs] = 60 * u
        v[row[at // bs], :, at % bs] = 0
    dt = torch.int8 if code == "int8" else torch.float8_e4m3fn
    k, v = k.to(dt), v.to(dt)
    ks, vs = torch.full((blocks, nkv), 1 / 60), torch.full((blocks, nkv), 1 / 64)
    c = kv.KVCache.from_buffers(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    T = sum(new)
    q = (u.repeat_interleave(nq // nkv, 0) + 0.1 * torch.randn((T, nq, d), generator=g)).to(R.DT[dtype])
    cu, scale = np.concatenate(([0], np.cumsum(new))).tolist(), float(np.float32(depth / d))
    mb = max(len(t) for t in table)
    out, lse = c.attend(q.cuda(), ints([t + [-1] * (mb - len(t)) for t in table]), ints(lens), ints(cu), scale=scale,
                        max_new=max(new), return_lse=True)
    want, wl = R.attend(q, k.float(), v.float(), ks, vs, table, lens, cu, scale)
    e = rel(out, want)
    print(f"dominant key {code} {dtype} d {d} new {new}: rel-L2 {e:.2e}")
    assert e <= REL[dtype] + (0.0 if dtype == "f32" else 2.0 ** -11), e
    assert (lse.cpu().double() - wl).abs().max().item() <= 2e-5


def test_a_new_cache_on_another_stream(kv):
    """A cache made and used on a side stream while the default stream is busy, 20 times over memory
    that the caches before it have used: its join counts are zeroed before its first call."""
    c, *_ = cache_of(kv, "int8", 300, 2, 64, 128)
    k, v, ks, vs = c.k, c.v, c.k_scale, c.v_scale
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((2, 16, 128), generator=g, device="cuda")
    args = (q, ints([list(range(0, 150)), list(range(150, 300))]), ints([9500, 9000]), ints([0, 1, 2]))
    want = c.attend(*args)
    busy = torch.randn((4096, 4096), device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(20):
        for _ in range(5):
            busy = (busy @ busy).clamp_(-1, 1)
        with torch.cuda.stream(s):
            other = kv.KVCache.from_buffers(k, v, ks, vs)
            got = other.attend(*args)
        s.synchronize()
        assert torch.equal(got, want), i
        other.check()
        other.close()


def test_attend_on_several_streams_at_once(kv):
    """Long contexts (whose pieces are joined through a workspace) on several streams of one cache at
    the same time, beside graphs that two streams captured: bit for bit what one call alone gives."""
    c, *_ = cache_of(kv, "int8", 400, 2, 64, 128)
    g = torch.Generator(device="cuda").manual_seed(4)
    cases = []
    for i in range(4):
        q = torch.randn((2 + 100 * (i == 3), 16, 128), generator=g, device="cuda")
        tab = ints([list(range(i, 180 + i)), list(range(200 - i, 380 - i))])
        lens, cu = ints([11500 - 700 * i, 9000]), ints([0, 1, q.shape[0]])
        cases.append((q, tab, lens, cu))
    want = [c.attend(*a) for a in cases]
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], []
    for a, s in zip(cases[:2], streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(c.attend(*a))
        graphs.append(graph)
    replayers = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for i in range(30):
        got = [c.attend(*cases[(i + j) % 4], stream=s) for j, s in enumerate(streams)]
        for graph, s in zip(graphs, replayers):
            with torch.cuda.stream(s):
                graph.replay()
        here = c.attend(*cases[i % 4])
        torch.cuda.synchronize()
        for j, x in enumerate(got):
            assert torch.equal(x, want[(i + j) % 4]), (i, j)
        assert torch.equal(here, want[i % 4]) and all(torch.equal(x, w) for x, w in zip(outs, want))
    c.check()


def test_attend_on_more_streams_than_workspaces(kv):
    """Streams that come and go, through the C entry: more than a cache keeps workspaces for, some
    destroyed so that their handles are used again."""
    import ctypes as C

    from rusty_engine_b200 import _lib

    c, *_ = cache_of(kv, "int8", 200, 2, 64, 128)
    q, out = torch.randn((2, 16, 128), device="cuda"), torch.zeros((2, 16, 128), device="cuda")
    tab, lens, cu = ints([list(range(0, 90)), list(range(100, 190))]), ints([5700, 5000]), ints([0, 1, 2])
    want = c.attend(q, tab, lens, cu)
    rows = lambda t: (t.data_ptr(), 16 * 128, 128, 16, 0)  # noqa: E731
    args = _lib.KV_ATTEND_ARGS.pack(*rows(q), *rows(out), tab.data_ptr(), lens.data_ptr(), cu.data_ptr(), 0, 2, 90, 2,
                                    0, float(np.float32(1 / np.sqrt(128))), 0, 1, 0)
    rt = C.CDLL("libcudart.so.12")
    torch.cuda.synchronize()
    kept = []
    for i in range(150):
        h = C.c_void_p()
        assert rt.cudaStreamCreateWithFlags(C.byref(h), 1) == 0
        assert _lib.load().rmoe_kv_attend(c._h, args, h) == _lib.RMOE_OK, _lib.load().rmoe_last_error()
        assert rt.cudaStreamSynchronize(h) == 0
        assert torch.equal(out, want), i
        out.zero_()
        torch.cuda.synchronize()
        if i % 3:
            kept.append(h)
        else:
            assert rt.cudaStreamDestroy(h) == 0
    for h in kept:
        assert rt.cudaStreamDestroy(h) == 0
    c.check()


def test_errors_right_after_a_check_are_kept(kv):
    """Errors on a stream that does not wait for the default one, each met right after the check that
    cleared the one before."""
    from rusty_engine_b200._lib import RmoeError

    c, rope = kv.KVCache(2, 16, 1, 64), kv.Rope(kv.RopeConfig(64), 10)
    x, far = torch.randn((1, 1, 64), device="cuda"), ints([64])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(50):
        with torch.cuda.stream(s):
            c.append(x, x, far)
            rope.apply(x, far)
        with pytest.raises(RmoeError, match="out of range"):
            c.check()
        with pytest.raises(RmoeError, match="position"):
            rope.check()
    c.check()
    rope.check()


def test_attend_is_right_again_after_a_lost_wait(kv):
    """Counts that a call left behind whose waits ran out: reported by check(), and gone after it."""
    from rusty_engine_b200 import _lib

    c, *_ = cache_of(kv, "int8", 400, 2, 64, 128)
    q = torch.randn((2, 16, 128), device="cuda")
    args = (q, ints([list(range(0, 180)), list(range(200, 380))]), ints([11500, 9000]), ints([0, 1, 2]))
    s = torch.cuda.Stream()
    want = c.attend(*args)
    torch.cuda.synchronize()
    assert torch.equal(c.attend(*args, stream=s), want)
    for _ in range(2):
        assert _lib.load().rmoe_selftest_kv_lost_wait(c._h) == _lib.RMOE_OK
        with pytest.raises(_lib.RmoeError, match="bounded wait"):
            c.check()
        got = c.attend(*args), c.attend(*args, stream=s), c.attend(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
        c.check()


# ---- handles ------------------------------------------------------------------------------------
def test_a_closed_rope_is_refused(kv):
    """Not taken for "no rope", which would write the keys unturned."""
    c = kv.KVCache(2, 16, 1, 64)
    rope = kv.Rope(kv.RopeConfig(64), 32)
    x, slots = torch.randn((3, 1, 64), device="cuda"), ints([0, 1, 2])
    rope.close()
    before = c.k.clone()
    for call in (lambda: c.append(x, x, slots, rope=rope, positions=slots), lambda: rope.apply(x, slots),
                 lambda: c.append(x, x, slots, rope=rope, positions=slots, q=x)):
        with pytest.raises(kv.EngineError, match="closed"):
            call()
    assert torch.equal(c.k, before)
    c.close()
    for call in (lambda: c.append(x, x, slots), lambda: c.read(slots), lambda: c.attend(x, ints([[0]]), ints([3]), ints([0, 3]))):
        with pytest.raises(kv.EngineError, match="closed"):
            call()


def test_return_lse_takes_any_truth_value(kv):
    c, *_ = cache_of(kv, "int8", 4, 2, 16, 64)
    q = torch.randn((2, 4, 64), device="cuda")
    for yes in (True, 1, np.True_):
        out, lse = c.attend(q, ints([[0, 1]]), ints([20]), ints([0, 2]), return_lse=yes)
        assert out.shape == q.shape and lse.shape == (2, 4)
    for no in (False, 0, np.False_, None):
        assert c.attend(q, ints([[0, 1]]), ints([20]), ints([0, 2]), return_lse=no).shape == q.shape


# ---- windows ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 7])
def test_attend_window_near_the_largest_integer(kv, dtype, window):
    """More queries than cached tokens (positions below 0) under windows that mean "all keys"."""
    run_attend(kv, "int8", dtype, [3, 40], [10, 5], 16, 8, 2, 64, window=window)
    run_attend(kv, "int8", dtype, [3], [12], 16, 4, 2, 256, window=window)
    run_attend(kv, "int8", dtype, [3, 200, 0], [300, 280, 90], 16, 16, 8, 64, window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new,bs,nq,nkv,d,window", [
    ([700, 300], [1, 1], 16, 8, 2, 128, 100), ([700], [3], 16, 4, 1, 64, 55), ([700], [1], 16, 4, 1, 256, 55),
    ([700], [40], 64, 4, 1, 256, 90), ([900], [300], 16, 32, 8, 128, 100), ([900], [300], 64, 32, 8, 64, 33)])
def test_attend_blocks_before_the_window_may_be_gone(kv, dtype, lens, new, bs, nq, nkv, d, window):
    """A server that gives blocks behind a sliding window back: entries of -1 (and beyond the cache)
    that no query sees change nothing and are no error; one inside the window is."""
    from rusty_engine_b200._lib import RmoeError

    blocks = sum(-(-n // bs) for n in lens) + 1
    c, *_ = cache_of(kv, "e4m3", blocks, nkv, bs, d)
    _, _, table = slots_of(lens, [0] * len(lens), bs, blocks)
    mb = max(len(t) for t in table)
    full = ints([t + [-1] * (mb - len(t)) for t in table])
    first = [max(0, n - m - window + 1) // bs for n, m in zip(lens, new)]
    holes = full.clone()
    for r, f in enumerate(first):
        assert f > 0
        holes[r, :f] = -1
        holes[r, 0] = blocks + 5
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn((sum(new), nq, d), generator=g, device="cuda").to(R.DT[dtype])
    call = lambda t: c.attend(q, t, ints(lens), ints(np.concatenate(([0], np.cumsum(new))).tolist()), window=window,  # noqa: E731
                              max_new=max(new), return_lse=True)
    want, wl = call(full)
    c.check()
    got, gl = call(holes)
    c.check()
    assert torch.equal(got, want) and torch.equal(gl, wl)
    holes[0, first[0]] = -1
    call(holes)
    with pytest.raises(RmoeError, match="out of range"):
        c.check()


# ---- scales -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("big", [1.0, 1e10, 1e14])
@pytest.mark.parametrize("lens,new,nq,nkv,d", [([200, 130], [1, 1], 8, 2, 128), ([180], [9], 4, 1, 256), ([700], [200], 32, 8, 64)])
def test_attend_blocks_of_zeros_beside_large_values(kv, dtype, big, lens, new, nq, nkv, d):
    """Blocks whose keys or values are all 0 (their scale is 0) keep their share of every row,
    however large the other blocks' values are."""
    bs = 16
    blocks = sum(-(-n // bs) for n in lens)
    c = kv.KVCache(blocks, bs, nkv, d)
    slots, _, table = slots_of(lens, lens, bs, blocks)
    g = torch.Generator().manual_seed(1)
    T = len(slots)
    k, v = torch.randn((T, nkv, d), generator=g), torch.randn((T, nkv, d), generator=g) * big
    pos = torch.cat([torch.arange(n) for n in lens])
    v[pos // bs % 3 == 0] = 0  # the first block too
    k[pos // bs % 4 == 1] = 0
    c.append(k.cuda(), v.cuda(), ints(slots))
    assert (c.v_scale == 0).any() and (c.k_scale == 0).any()
    q = torch.randn((sum(new), nq, d), generator=g).to(R.DT[dtype])
    cu = np.concatenate(([0], np.cumsum(new))).tolist()
    mb = max(len(t) for t in table)
    out, lse = c.attend(q.cuda(), ints([t + [-1] * (mb - len(t)) for t in table]), ints(lens), ints(cu), max_new=max(new),
                        return_lse=True)
    want, wl = R.attend(q, c.k.cpu().float(), c.v.cpu().float(), c.k_scale.cpu(), c.v_scale.cpu(), table, lens, cu,
                        float(np.float32(1 / np.sqrt(d))))
    assert rel(out, want) <= REL[dtype]
    assert (lse.cpu().double() - wl).abs().max().item() <= 2e-5
    c.check()


def test_batch_step_in_a_cuda_graph_moves_on(kv):
    """KVBatch.extend, append, attend and release captured once: every replay is the next step."""
    b, e = kv.KVBatch(3, 8, 20, 16), kv.KVBatch(3, 8, 20, 16)
    caches = [kv.KVCache(20, 16, 2, 64) for _ in (b, e)]
    x = torch.randn((3, 8, 64), device="cuda")
    done, new = ints([0, 0, 0]), ints([1, 1, 1])

    def step(batch, c):
        st = batch.extend(new, 3)
        c.append(x[:, 4:6], x[:, 6:], st.slots)
        out = c.attend(x[:, :4], batch.table, batch.lens, st.cu, max_new=1)
        batch.release(done)
        return out

    first = ints([15, 0, 30])
    for batch, c in zip((b, e), caches):
        st = batch.extend(first, 45)
        c.append(torch.ones((45, 2, 64), device="cuda"), torch.ones((45, 2, 64), device="cuda"), st.slots)
        step(batch, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(b, caches[0])
    for i in range(20):
        x.copy_(torch.randn((3, 8, 64), device="cuda"))
        done.copy_(ints([int(i == 7), 0, int(i == 11)]))
        g.replay()
        want = step(e, caches[1])
        assert torch.equal(out, want), i
        assert b.lens.tolist() == e.lens.tolist() and b.n_free.tolist() == e.n_free.tolist()
        assert torch.equal(b.table, e.table)
    assert b.lens.tolist() == [12, 21, 8]


def test_open_cache_positions_reach_as_far_as_its_blocks(kv):
    """max_pos inside a block: the table has room up to the block's end, and so has the rope."""
    from rusty_engine_b200.stack import MoEStack, make_block
    from test_stack import small_geometry

    geo = small_geometry()
    stack = MoEStack(geo, [make_block(geo, seed=3, dlo=0.001, dhi=0.004, attn_dlo=0.002, attn_dhi=0.01)], device=0)
    stack.open_cache(max_requests=1, n_blocks=4, block_size=16, max_pos=20)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((32, geo.d_model), generator=g, device="cuda")
    stack.step(x, ints([32]), max_new=32)
    assert stack.batch.lens.tolist() == [32]  # the table takes them
    stack.caches[0].check()                   # and every position is turned
    stack.close()


# ---- many requests, many runs -------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reqs", [33, 40, 257, 300, 600])
def test_attend_many_requests(kv, dtype, reqs):
    """More requests than a warp's lanes, than the split kernel's threads and than the prompt
    kernel's; empty ones among them; then the same beside prompts for the prompt kernel."""
    rng = np.random.default_rng(reqs)
    lens = rng.integers(0, 70, reqs).tolist()
    new = [int(min(n, m)) for n, m in zip(rng.integers(0, 4, reqs), lens)]
    run_attend(kv, "int8", dtype, lens, new, 16, 2, 1, 64)
    run_attend(kv, "e4m3", dtype, lens, [min(n, 1) for n in lens], 32, 6, 2, 128, window=9)
    for r, (n, m) in zip((reqs - 1, 0, reqs // 2), ((300, 260), (270, 270), (200, 130))):
        lens[r], new[r] = n, m
    run_attend(kv, "int8", dtype, lens, new, 16, 16, 8, 64)
    run_attend(kv, "int8", dtype, lens, new, 64, 16, 8, 64, max_new=False, pad=7, window=50)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("reqs", [1025, 1500])
def test_append_many_single_tokens(kv, code, bs, reqs):
    """More than 1024 runs of one token each, some slots skipped."""
    rng = np.random.default_rng(reqs + bs)
    c, k, v, ks, vs = cache_of(kv, code, reqs, 2, bs, 64)
    order = rng.permutation(reqs)
    slots = [int(b) * bs + int(rng.integers(0, bs)) if rng.random() < 0.9 else -1 for b in order]
    g = torch.Generator().manual_seed(7)
    kn, vn = (torch.randn((reqs, 2, 64), generator=g) * torch.rand((reqs, 1, 1), generator=g) * 4 for _ in "kv")
    c.append(kn.cuda(), vn.cuda(), ints(slots))
    R.append(k, ks, kn.numpy(), slots, bs, code)
    R.append(v, vs, vn.numpy(), slots, bs, code)
    assert np.array_equal(c.k_scale.cpu().numpy(), ks) and np.array_equal(c.v_scale.cpu().numpy(), vs)
    assert np.array_equal(c.k.float().cpu().numpy(), k) and np.array_equal(c.v.float().cpu().numpy(), v)
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,nq,strided", [(640, 32, False), (1300, 16, False), (1300, 16, True)])
def test_append_beside_the_rope_of_a_long_q(kv, dtype, T, nq, strided):
    """A q long enough for its own kernel, beside which the cache is written: inputs that the stream
    has just made, q in place, and attention right after, against the calls one by one, bit for bit."""
    rope = kv.Rope(kv.RopeConfig(128, 1e6), 4096)
    blocks = -(-T // 64)
    a, b = (kv.KVCache(blocks, 64, 2, 128) for _ in "ab")
    table, lens, cu = ints([list(range(blocks))]), ints([T]), ints([0, T])
    g = torch.Generator(device="cuda").manual_seed(5)
    for i in range(6):
        base = torch.randn((T, nq + 4 + strided, 128), generator=g, device="cuda").to(R.DT[dtype])
        pos = torch.arange(T, dtype=torch.int32, device="cuda")
        x, slots = base * 2, pos + 0
        q, k, v = x[:, :nq], x[:, nq:nq + 2], x[:, nq + 2:nq + 4]
        if not strided:
            q = q.contiguous()
        got = a.append(k, v, slots, rope=rope, positions=pos, q=q, q_out=q)
        out = a.attend(got, table, lens, cu, max_new=T)
        torch.cuda.synchronize()
        x = base * 2
        qr, kr = rope.apply(x[:, :nq], pos, x[:, nq:nq + 2])
        torch.cuda.synchronize()
        b.append(kr.float(), x[:, nq + 2:nq + 4].float(), slots)
        torch.cuda.synchronize()
        assert torch.equal(got, qr), i
        if dtype == "f32":  # (in 16 bits the keys would be rounded between rope and cache)
            for m, n in ((a.k, b.k), (a.k_scale, b.k_scale)):
                assert torch.equal(m, n), i
        assert torch.equal(a.v, b.v) and torch.equal(a.v_scale, b.v_scale)
        assert torch.equal(out, a.attend(qr, table, lens, cu, max_new=T))
    a.check()


def test_attend_on_new_streams_while_another_captures(kv):
    """A call that is captured and a plain one on another stream in the middle of the capture, each the
    first of its stream: the workspaces they need are made without ending the capture."""
    from rusty_engine_b200 import _lib

    c, *_ = cache_of(kv, "int8", 200, 2, 64, 128)
    q = torch.randn((2, 16, 128), device="cuda")
    outs = [torch.zeros_like(q) for _ in range(3)]
    tab, lens, cu = ints([list(range(0, 90)), list(range(100, 190))]), ints([5700, 5000]), ints([0, 1, 2])
    want = c.attend(q, tab, lens, cu)
    rows = lambda t: (t.data_ptr(), 16 * 128, 128, 16, 0)  # noqa: E731

    def call(out, stream):
        args = _lib.KV_ATTEND_ARGS.pack(*rows(q), *rows(out), tab.data_ptr(), lens.data_ptr(), cu.data_ptr(), 0, 2, 90, 2, 0,
                                        float(np.float32(1 / np.sqrt(128))), 0, 1, 0)
        assert _lib.load().rmoe_kv_attend(c._h, args, stream.cuda_stream) == _lib.RMOE_OK, _lib.load().rmoe_last_error()

    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        call(outs[0], streams[0])
        call(outs[1], streams[1])
        call(outs[2], streams[2])
        call(outs[0], streams[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[1], want) and torch.equal(outs[2], want) and not outs[0].any()
    for _ in range(3):
        outs[0].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)
    c.check()
