"""The paged 8-bit KV cache operators (rusty_engine_b200.kv) on the GPU, against tests/kv_ref.py.

Tolerances, from the operations and not from runs:
* tables, slots, positions and codes are whole numbers or defined float32 steps: equal.
* rope: two f32 products and a sum of values whose cos / sin are rounded once, at most 4 * 2^-24 of
  |x0| + |x1|, then the output's own rounding (2^-11 f16, 2^-8 bf16).
* attention: q and codes are exact as fp16 (pairs for f32), sums are f32.  f32: scores of up to
  about 20 are off by 20 * 2^-22, the probabilities by that and their pair's 2^-22, so rel-L2
  <= 1e-5.  f16 / bf16 calls round the probabilities to fp16 (2^-11) and the output to its type
  (2^-11 / 2^-8): rel-L2 <= 2^-10 and 2^-8 + 2^-11.  lse: 2e-5 absolute.
"""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu

REL = {"f32": 1e-5, "f16": 2.0 ** -10, "bf16": 2.0 ** -8 + 2.0 ** -11}
ULP = {"f32": 4 * 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def kv(gpu):
    from rusty_engine_b200 import kv as m

    return m


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def rel(got, want):
    d = (got.double().cpu() - want).norm()
    return float(d / want.norm()) if want.norm() > 0 else float(d)


# ---- extend / release ----------------------------------------------------------------------------
@pytest.mark.parametrize("reqs,bs,top_new,free_share,mb_extra,cut", [
    (1, 16, 1, 1.0, 0, 0), (1, 128, 700, 1.0, 2, 0), (7, 16, 40, 1.0, 0, 0), (40, 32, 65, 0.5, 1, 0),
    (33, 64, 1, 1.0, 0, 5), (700, 64, 300, 0.8, 0, -37), (1500, 16, 3, 1.0, 0, 0), (5, 16, 33, 0.0, 3, 0)])
def test_extend_matches_loops(kv, reqs, bs, top_new, free_share, mb_extra, cut):
    """Ragged, zero and negative new lengths, a pool that runs out, rows that overflow, a batch
    padded past its tokens (cut < 0) and one cut short of them (cut > 0)."""
    rng = np.random.default_rng(reqs * 1000 + bs)
    lens = rng.integers(0, 5 * bs, reqs).tolist()
    new = [int(v) for v in rng.integers(-1 if reqs > 5 else 1, top_new + 1, reqs)]
    have = [-(-x // bs) for x in lens]
    want = [-(-(x + max(n, 0)) // bs) for x, n in zip(lens, new)]
    mb = max(max(want) + mb_extra - (1 if reqs > 30 else 0), max(have), 1)
    order = rng.permutation(sum(want) + 9).tolist()
    table, at = [], 0
    for h in have:
        table.append(order[at:at + h] + [-1] * (mb - h))
        at += h
    free = order[at:]
    n_free = int(len(free) * free_share)
    total = sum(max(n, 0) for n in new) - cut
    t, l, f, nf = ints(table), ints(lens), ints(free), ints([n_free])
    st = kv.extend_tables(t, l, ints(new), f, nf, total, bs)
    w_table, cu, pos, slots, out, left = R.extend(table, lens, new, free, n_free, total, bs)
    assert st.cu.tolist() == cu and st.positions.tolist() == pos and st.slots.tolist() == slots
    assert st.lens.tolist() == out and st.n_free.tolist() == [left]
    assert t.tolist() == w_table
    assert l.tolist() == lens and nf.tolist() == [n_free]  # inputs stay


def test_batch_extend_release_cycle(kv):
    """Requests grow, end and are replaced; every block is held once or free, never both."""
    rng = np.random.default_rng(3)
    b = kv.KVBatch(6, 12, 40, 16)
    for i in range(30):
        new = rng.integers(0, 40, 6)
        b.extend(ints(new.tolist()), int(new.sum()))
        lens, tab, n = b.lens.tolist(), b.table.tolist(), int(b.n_free)
        held = [x for r in range(6) for x in tab[r][: -(-lens[r] // 16)]]
        assert sorted(held + b.free[:n].tolist()) == list(range(40))
        done = (rng.random(6) < 0.4).astype(int)
        b.release(ints(done.tolist()))
        assert all(not d or (b.lens[r] == 0 and (b.table[r] == -1).all()) for r, d in enumerate(done))
    assert b.extend(ints([0] * 6), 0).slots.numel() == 0


# ---- rope ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("d,rot,nq,nk,T", [(128, 128, 32, 4, 7), (64, 32, 3, 1, 1), (256, 256, 2, 2, 130),
                                           (80, 40, 5, 0, 9), (96, 24, 1, 1, 33), (128, 64, 8, 8, 1000), (128, 128, 6, 1, 1900),
                                           (64, 32, 5, 0, 3001), (256, 256, 3, 2, 1184)])
def test_rope_matches_float64(kv, dtype, half, d, rot, nq, nk, T):
    g = torch.Generator().manual_seed(T)
    cfg = kv.RopeConfig(rot, 1e6, kv.RopeLayout.Half if half else kv.RopeLayout.Interleaved)
    rope = kv.Rope(cfg, 131072)
    x = torch.randn((T, nq + nk + 1, d), generator=g).to(R.DT[dtype]).cuda()
    q, k = x[:, :nq], x[:, nq:nq + nk]  # views of one buffer
    pos = torch.randint(0, 131072, (T,), generator=g).tolist()
    f, m = R.frequencies(rot, 1e6)
    got = rope.apply(q, ints(pos), k if nk else None)
    got = got if nk else (got,)
    for a, b in zip(got, (q, k)):
        want = R.rope(b, pos, f, m, half)
        # each element of a pair: |y| <= |x0| + |x1|; a passed element is itself
        bound = ULP[dtype] * (b.double().cpu().abs().amax(dim=2, keepdim=True) * 2) + 4 * 2.0 ** -24 * 8
        assert ((a.double().cpu() - want).abs() <= bound).all()
        assert torch.equal(a[..., rot:], b[..., rot:])
    rope.check()


def test_rope_odd_strides_in_place_and_back(kv):
    """Misaligned views, turning in place and back again, against the aligned call bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rope = kv.Rope(kv.RopeConfig(64, 1e4, kv.RopeLayout.Half), 100)
    pos = ints(list(range(11)))
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.randn((11, 4 * 129 + 1), generator=g, device="cuda").to(dt)
        q = buf[:, 1:].view(11, 4, 129)[:, :, 1:]
        want = rope.apply(q.contiguous(), pos)
        assert torch.equal(rope.apply(q, pos), want)
        keep = q.clone()
        assert rope.apply(q, pos, out=q).data_ptr() == q.data_ptr() and torch.equal(q, want)
        back = rope.apply(want, pos, inverse=True)
        assert (back.float() - keep.float()).abs().max() < (1e-5 if dt == torch.float32 else 0.1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rope_long_batches_in_place(kv, dtype):
    """Long batches take another kernel: in place on views of a fused buffer, whose other heads stay,
    against the same tokens in short batches bit for bit; a position outside leaves its token alone."""
    from rusty_engine_b200._lib import RmoeError

    g = torch.Generator(device="cuda").manual_seed(1)
    rope = kv.Rope(kv.RopeConfig(64, 1e4, kv.RopeLayout.Interleaved), 5000)
    x = torch.randn((2500, 4 + 2 + 2, 128), generator=g, device="cuda").to(R.DT[dtype])
    pos = torch.randint(0, 5000, (2500,), generator=g, device="cuda").to(torch.int32)
    pos[7], pos[2400] = 5000, -3
    keep = x.clone()
    want = [rope.apply(x[i:i + 500, :4], pos[i:i + 500], x[i:i + 500, 4:6]) for i in range(0, 2500, 500)]
    q, k = (torch.cat(w) for w in zip(*want))
    rope.apply(x[:, :4], pos, x[:, 4:6], out=x[:, :4], k_out=x[:, 4:6])
    assert torch.equal(x[:, :4], q) and torch.equal(x[:, 4:6], k) and torch.equal(x[:, 6:], keep[:, 6:])
    assert torch.equal(x[7], keep[7]) and torch.equal(x[2400], keep[2400])
    with pytest.raises(RmoeError, match="position"):
        rope.check()


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="yarn", factor=4.0, orig=4096),
                                dict(scaling="yarn", factor=40.0, orig=4096, fast=32.0, slow=2.0),
                                dict(ff=[1.0 + 0.25 * i for i in range(32)])])
def test_rope_scaled_tables(kv, kw):
    """cos and sin of every scaling at long positions, read out by turning unit vectors."""
    name = {"none": kv.RopeScaling.NoScaling, "linear": kv.RopeScaling.Linear, "yarn": kv.RopeScaling.Yarn}
    cfg = kv.RopeConfig(64, 1e4, kv.RopeLayout.Half, name[kw.get("scaling", "none")], kw.get("factor", 1.0),
                        kw.get("orig", 0), kw.get("fast", 32.0), kw.get("slow", 1.0), freq_factors=kw.get("ff"))
    rope = kv.Rope(cfg, 200000)
    pos = [0, 1, 4095, 65537, 199999]
    x = torch.zeros((5, 1, 64), device="cuda")
    x[..., :32] = 1.0
    f, m = R.frequencies(64, 1e4, **kw)
    got = rope.apply(x, ints(pos)).cpu().double()
    a = np.asarray(pos, dtype=np.float64)[:, None] * f
    want = torch.from_numpy(np.concatenate((m * np.cos(a), m * np.sin(a)), axis=1))[:, None]
    assert (got - want).abs().max() <= 2.0 ** -24 * m + 1e-9  # one rounding each


def test_rope_position_outside_is_reported(kv):
    from rusty_engine_b200._lib import RmoeError

    rope = kv.Rope(kv.RopeConfig(64), 10)
    x = torch.randn((3, 1, 64), device="cuda")
    y = rope.apply(x, ints([0, 10, -1]))
    assert torch.equal(y, x)  # position 0 turns by nothing, the others are left alone
    with pytest.raises(RmoeError, match="position"):
        rope.check()
    rope.check()


# ---- append / read -------------------------------------------------------------------------------
def cache_of(kv, code, blocks, heads, bs, d, seed=0):
    """A cache with random codes and scales, and its values as float32 numbers on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((blocks, heads, bs, d), generator=g)
    codes = lambda y: (y * 30).round().clamp(-127, 127).to(torch.int8) if code == "int8" else (y * 90).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    k, v = codes(x), codes(x.flip(0) * 0.7)
    ks = (torch.rand((blocks, heads), generator=g) + 0.5) / 30
    vs = (torch.rand((blocks, heads), generator=g) + 0.5) / 30
    c = kv.KVCache.from_buffers(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    return c, k.float().numpy(), v.float().numpy(), ks.numpy(), vs.numpy()


def slots_of(lens, new, bs, blocks, seed=0):
    """(slots, positions, table) of requests that hold lens - new tokens and add new."""
    order = np.random.default_rng(seed).permutation(blocks).tolist()
    slots, pos, table, at = [], [], [], 0
    for n, m in zip(lens, new):
        row = order[at:at - (-n // bs)]
        at += -(-n // bs)
        table.append(row)
        for p in range(n - m, n):
            slots.append(row[p // bs] * bs + p % bs)
            pos.append(p)
    return slots, pos, table


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,new,bs,heads,d", [
    ([1], [1], 16, 1, 64), ([17, 33, 5], [1, 1, 1], 16, 4, 128), ([130, 1, 64], [130, 1, 17], 64, 2, 128),
    ([300], [255], 128, 1, 256), ([40, 41, 42, 43], [3, 0, 42, 9], 32, 3, 64), ([2500], [2177], 64, 1, 128)])
def test_append_codes_equal(kv, code, dtype, lens, new, bs, heads, d):
    """Codes and scales bit for bit, with blocks that already hold tokens (whose codes are rounded
    again where the scale grows) and blocks with stale content; then read() of every slot."""
    blocks = sum(-(-n // bs) for n in lens) + 2
    c, k, v, ks, vs = cache_of(kv, code, blocks, heads, bs, d, seed=len(lens))
    slots, _, _ = slots_of(lens, new, bs, blocks)
    g = torch.Generator().manual_seed(7)
    T = len(slots)
    kn = (torch.randn((T, heads, d), generator=g) * torch.rand((T, 1, 1), generator=g) * 4).to(R.DT[dtype])
    vn = torch.randn((T, heads, d), generator=g).to(R.DT[dtype])
    vn[::3] = 0
    assert c.append(kn.cuda(), vn.cuda(), ints(slots)) is None
    R.append(k, ks, kn.float().numpy(), slots, bs, code)
    R.append(v, vs, vn.float().numpy(), slots, bs, code)
    assert np.array_equal(c.k_scale.cpu().numpy(), ks) and np.array_equal(c.v_scale.cpu().numpy(), vs)
    assert np.array_equal(c.k.float().cpu().numpy(), k) and np.array_equal(c.v.float().cpu().numpy(), v)
    every = [-1] + list(range(blocks * bs))
    for dt in (torch.float32, torch.bfloat16):
        gk, gv = c.read(ints(every), dt)
        for got, val, sc in ((gk, k, ks), (gv, v, vs)):
            want = torch.from_numpy((val * sc[:, :, None, None]).transpose(0, 2, 1, 3).reshape(-1, heads, d)).to(dt)
            assert torch.equal(got[1:].cpu(), want) and not got[0].any()
    c.check()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rot", [128, 48])
def test_append_with_rope_is_rope_then_append(kv, half, rot):
    """The fused call against rope.apply and a plain append, bit for bit (f32), q included, on
    strided views and in place."""
    cfg = kv.RopeConfig(rot, 1e6, kv.RopeLayout.Half if half else kv.RopeLayout.Interleaved)
    rope = kv.Rope(cfg, 4096)
    lens, new = [100, 3, 700], [37, 3, 1]
    slots, pos, _ = slots_of(lens, new, 32, 40)
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn((len(slots), 12 + 2 + 2, 128), generator=g, device="cuda")
    q, k, v = qkv[:, :12], qkv[:, 12:14], qkv[:, 14:]
    a, *_ = cache_of(kv, "int8", 40, 2, 32, 128)
    b, *_ = cache_of(kv, "int8", 40, 2, 32, 128)
    qr, kr = rope.apply(q, ints(pos), k)
    a.append(kr, v, ints(slots))
    got = b.append(k, v, ints(slots), rope=rope, positions=ints(pos), q=q)
    assert torch.equal(got, qr)
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        assert torch.equal(x, y)
    assert b.append(k, v, ints(slots), rope=rope, positions=ints(pos), q=q, q_out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, qr) and torch.equal(a.k, b.k)


def test_append_edges(kv):
    """Zeros, values too small for a normal scale, the largest floats, skipped and foreign slots,
    NaN and infinities (stored as 0 and the largest code, and reported)."""
    from rusty_engine_b200._lib import RmoeError

    for code in ("int8", "e4m3"):
        top = 127.0 if code == "int8" else 448.0
        c, k, v, ks, vs = cache_of(kv, code, 4, 1, 16, 64)
        x = torch.zeros((6, 1, 64))
        x[1] = 1e-42
        x[2] = 3e38
        x[3, 0, :3] = torch.tensor([-1.0, 0.5, 1.0])
        x[4] = 5.0
        slots = [0, 1, 2, 16, -1, 35]  # one run of three, a block of its own, skipped, the middle of a block
        R.append(k, ks, x.numpy()[:, :], slots, 16, code)
        R.append(v, vs, x.numpy()[:, :], slots, 16, code)
        c.append(x.cuda(), x.cuda(), ints(slots))
        assert np.array_equal(c.k.float().cpu().numpy(), k) and np.array_equal(c.k_scale.cpu().numpy(), ks)
        c.check()
        x[3, 0, 3:6] = torch.tensor([float("nan"), float("inf"), -float("inf")])
        c.append(x[3:4].cuda(), x[:1].cuda(), ints([16]))
        assert c.k[1, 0, 0, :6].float().tolist()[3:] == [0.0, top, -top] and float(c.k_scale[1, 0]) == np.float32(1) / np.float32(top)
        with pytest.raises(RmoeError, match="not finite"):
            c.check()
        before = c.k.view(torch.uint8).clone()
        c.append(x[:1].cuda(), x[:1].cuda(), ints([64]))  # past the last block
        assert torch.equal(before, c.k.view(torch.uint8))
        with pytest.raises(RmoeError, match="out of range"):
            c.check()
        c.append(x[:0].cuda(), x[:0].cuda(), ints([]))
        c.check()


# ---- attend --------------------------------------------------------------------------------------
def run_attend(kv, code, dtype, lens, new, bs, nq, nkv, d, window=0, scale=None, pad=0, max_new=True, poison=False, seed=0,
               far=0.0):
    blocks = sum(-(-max(n, 0) // bs) for n in lens) + 3
    c, k, v, ks, vs = cache_of(kv, code, blocks, nkv, bs, d, seed=seed)
    _, _, table = slots_of([max(n, 0) for n in lens], [0] * len(lens), bs, blocks)
    g = torch.Generator().manual_seed(seed + 1)
    T = sum(new) + pad
    q = (2 * torch.randn((T, nq, d), generator=g)).to(R.DT[dtype])
    cu = np.concatenate(([0], np.cumsum(new))).tolist()
    if poison:  # what lies past each request's end must not be seen: the codes' extremes, NaN in e4m3
        raw = c.k.view(torch.uint8), c.v.view(torch.uint8)
        for r, n in enumerate(lens):
            if n % bs:
                for x in raw:
                    x[table[r][-1], :, n % bs:] = 0x7F if code == "e4m3" else 0x80
    mb = max(1, max(len(t) for t in table)) + 1
    tab = ints([t + [-1] * (mb - len(t)) for t in table])
    scale = 1 / np.sqrt(d) if scale is None else scale
    out, lse = c.attend(q.cuda(), tab, ints(lens), ints(cu), scale=scale, window=window,
                        max_new=max(new) if max_new else None, return_lse=True)
    c.check()
    want, wl = R.attend(q, k, v, ks, vs, table, lens, cu, float(np.float32(scale)), window)
    assert out.dtype == q.dtype and torch.isfinite(out.float()).all()
    e = rel(out, want)
    print(f"attend {code} {dtype} lens {lens[:4]} new {new[:4]}: rel-L2 {e:.2e}")
    hidden = torch.isinf(wl)
    loose = far * float(wl[~hidden].abs().max()) if far else 0.0
    assert e <= REL[dtype] + loose, e
    hidden = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse.cpu()), hidden) and not out.cpu()[hidden].any()
    assert (lse.cpu().double() - wl)[~hidden].abs().max().item() <= 2e-5 + loose if (~hidden).any() else True


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,new,bs,nq,nkv,d", [
    ([1], [1], 16, 1, 1, 64), ([97], [1], 16, 32, 4, 128), ([15, 16, 17, 1], [1, 1, 1, 1], 16, 8, 1, 128),
    ([63, 64, 65, 129, 1000], [1, 1, 1, 2, 1], 64, 10, 2, 64), ([700, 3], [3, 3], 128, 6, 3, 256),
    ([2049, 31], [1, 1], 32, 20, 4, 128)])
def test_attend_decode(kv, code, dtype, lens, new, bs, nq, nkv, d):
    run_attend(kv, code, dtype, lens, new, bs, nq, nkv, d, seed=len(lens))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,new,bs,nq,nkv,d", [
    ([150], [150], 16, 8, 1, 128), ([300, 7, 129], [77, 7, 129], 64, 4, 2, 64), ([257], [200], 128, 2, 2, 256),
    ([129, 90, 260], [129, 1, 130], 32, 16, 2, 128), ([1000], [333], 64, 5, 1, 128)])
def test_attend_prompts(kv, code, dtype, lens, new, bs, nq, nkv, d):
    run_attend(kv, code, dtype, lens, new, bs, nq, nkv, d, seed=len(lens))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,new,bs,nq,nkv,d,window", [
    ([300], [300], 16, 32, 8, 128, 0), ([520, 7, 140, 0], [300, 1, 140, 0], 64, 16, 8, 64, 0),
    ([129, 700], [128, 129], 128, 40, 8, 128, 0), ([70, 90, 64, 33], [64, 64, 64, 33], 32, 8, 8, 64, 0),
    ([600, 40], [257, 40], 64, 24, 8, 128, 100), ([400, 300], [140, 1], 16, 48, 12, 128, 33)])
def test_attend_prompts_of_many_rows(kv, code, dtype, lens, new, bs, nq, nkv, d, window):
    """Enough rows for the tensor-core prompt kernel (24 CTAs of 256 rows), beside short requests."""
    run_attend(kv, code, dtype, lens, new, bs, nq, nkv, d, window=window, seed=len(lens))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_many_rows_edges(kv, code, dtype):
    """The prompt kernel's rows that see nothing, garbage past the ends, scores near to each other,
    and repeats bit for bit."""
    run_attend(kv, code, dtype, [3, 200, 0], [300, 280, 90], 16, 16, 8, 64, pad=50, poison=True, max_new=False)
    run_attend(kv, code, dtype, [190, 333], [190, 150], 64, 16, 8, 128, pad=3, poison=True)
    run_attend(kv, code, dtype, [700], [200], 64, 32, 8, 64, scale=0.001)
    c, *_ = cache_of(kv, code, 40, 8, 64, 128)
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((500, 32, 128), generator=g, device="cuda").to(R.DT[dtype])
    args = (ints([list(range(0, 20)), list(range(20, 40))]), ints([1200, 900]), ints([0, 300, 500]))
    a, b = c.attend(q, *args), c.attend(q, *args)
    assert torch.equal(a, b)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 33])
@pytest.mark.parametrize("lens,new,bs,nq,nkv,d", [
    ([200], [200], 16, 4, 2, 256), ([333, 40], [77, 40], 32, 3, 3, 256), ([150], [9], 64, 1, 1, 256),
    ([90, 0, 61], [17, 3, 50], 16, 8, 4, 256), ([500], [24], 64, 5, 1, 64), ([260, 7], [12, 7], 16, 12, 4, 128)])
def test_attend_prompts_on_split_keys(kv, code, dtype, window, lens, new, bs, nq, nkv, d):
    """Even and odd numbers of row tiles, whose early rows see few of the keys."""
    run_attend(kv, code, dtype, lens, new, bs, nq, nkv, d, window=window, seed=sum(new), poison=True)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_scores_in_the_hundreds(kv, code, dtype):
    """Scores so far apart that the maximum grows from tile to tile.  A score of size s is a sum of
    128 products whose running sums the tensor cores cut to 24 bits at most 16 times, and is rounded
    three more times at 1.44 s: off by at most 2^-19 s, and so are lse and, relatively, the weights."""
    run_attend(kv, code, dtype, [700], [200], 64, 32, 8, 128, scale=1.0, far=2.0 ** -19)
    run_attend(kv, code, dtype, [700, 90], [1, 2], 64, 32, 8, 128, scale=1.0, far=2.0 ** -19)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000000])
@pytest.mark.parametrize("lens,new", [([300, 40], [1, 1]), ([300, 77], [150, 77])])
def test_attend_window(kv, dtype, window, lens, new):
    run_attend(kv, "int8", dtype, lens, new, 64, 8, 2, 128, window=window)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new", [([0, 5, 0], [1, 1, 0]), ([2, 40], [5, 3]), ([0], [4]), ([3, 200], [140, 150])])
def test_attend_rows_that_see_nothing(kv, code, dtype, lens, new):
    """Empty requests, more queries than tokens, padding tokens: 0 and -infinity; garbage past the
    requests' ends, NaN codes among it, stays unseen."""
    run_attend(kv, code, dtype, lens, new, 16, 8, 2, 64, pad=3, poison=True)
    run_attend(kv, code, dtype, lens, new, 64, 4, 4, 128, pad=200, poison=True, max_new=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.001])
def test_attend_scales(kv, dtype, scale):
    """Scores spread so far that a row is one key, and so little that it is a mean."""
    run_attend(kv, "int8", dtype, [500], [1], 64, 8, 1, 128, scale=scale)
    run_attend(kv, "int8", dtype, [200], [130], 64, 8, 1, 128, scale=scale)


@pytest.mark.parametrize("size", [1e-4, 3e4])
def test_attend_large_and_small_queries(kv, size):
    """q far from 1 (beyond fp16's own range for the products of f32 and bf16): the rows' scale
    carries it."""
    for dtype in ("f32", "bf16"):
        c, k, v, ks, vs = cache_of(kv, "int8", 8, 1, 16, 128)
        g = torch.Generator().manual_seed(2)
        q = (torch.randn((140, 4, 128), generator=g) * size * 30).to(R.DT[dtype])
        table, lens, cu = [[3, 1, 7, 0, 2]], [75], [0, 140]
        for rows in (1, 140):
            want, _ = R.attend(q[:rows], k, v, ks, vs, table, [75], [0, rows], float(np.float32(0.1 / size / 30)))
            out = c.attend(q[:rows].cuda(), ints(table), ints(lens), ints([0, rows]), scale=0.1 / size / 30)
            assert rel(out, want) <= REL[dtype]


def test_attend_strided_views_and_stream(kv):
    """Views of a fused buffer, misaligned ones, an output view, another stream: as the plain call."""
    c, *_ = cache_of(kv, "int8", 12, 2, 32, 128)
    tab, lens, cu = ints([[0, 5, 2], [7, 9, 1]]), ints([70, 90]), ints([0, 1, 41])
    g = torch.Generator(device="cuda").manual_seed(2)
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.randn((41, 8 * 131 + 5), generator=g, device="cuda").to(dt)
        q = buf[:, 3:3 + 8 * 131].view(41, 8, 131)[:, :, 1:129]
        want = c.attend(q.contiguous(), tab, lens, cu)
        assert torch.equal(c.attend(q, tab, lens, cu), want)
        wide = torch.zeros((41, 9, 256), dtype=dt, device="cuda")
        c.attend(q, tab, lens, cu, out=wide[:, 1:, 64:192])
        assert torch.equal(wide[:, 1:, 64:192], want) and not wide[:, 0].any() and not wide[..., :64].any()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        other = c.attend(q, tab, lens, cu, stream=s)
        s.synchronize()
        assert torch.equal(other, want)


def test_attend_repeats_bit_for_bit(kv):
    """The same call twice, on long contexts split over the chip and in a mixed batch: equal bits."""
    c, *_ = cache_of(kv, "int8", 400, 2, 64, 128)
    tab = ints([list(range(0, 180)), list(range(200, 380))])
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((300, 16, 128), generator=g, device="cuda")
    for cu, lens in (([0, 1, 2], [11500, 9000]), ([0, 1, 300], [11000, 400])):
        a = c.attend(q[:cu[-1]], tab, ints(lens), ints(cu), return_lse=True)
        b = c.attend(q[:cu[-1]], tab, ints(lens), ints(cu), return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attend_foreign_blocks_are_reported(kv):
    """Table entries outside the cache are skipped and reported, never read."""
    from rusty_engine_b200._lib import RmoeError

    c, k, v, ks, vs = cache_of(kv, "int8", 6, 1, 16, 64)
    q = torch.randn((2, 4, 64), device="cuda")
    out = c.attend(q, ints([[2, 6, 1], [0, -1, 3]]), ints([48, 48]), ints([0, 1, 2]))
    assert torch.isfinite(out).all()
    with pytest.raises(RmoeError, match="out of range"):
        c.check()


def test_attend_far_blocks(kv):
    """Codes whose byte offset is beyond 2^32: the last blocks of a 5 GB cache."""
    n, d, bs = 5 * 2 ** 30 // (128 * 128), 128, 128
    k = torch.zeros((n, 1, bs, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((n, 1, bs, d), dtype=torch.int8, device="cuda")
    s = torch.full((n, 1), 0.02, device="cuda")
    c = kv.KVCache.from_buffers(k, v, s, s.clone())
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((200, 1, d), generator=g, device="cuda")
    blocks = [n - 1, n - 7]
    slots = [blocks[p // bs] * bs + p % bs for p in range(200)]
    c.append(x, x, ints(slots))
    gk, _ = c.read(ints(slots))
    assert (gk - x).abs().max() <= x.abs().max() / 127
    for rows in (1, 200):
        q = torch.randn((rows, 2, d), generator=g, device="cuda")
        out = c.attend(q, ints([blocks]), ints([200]), ints([0, rows]))
        want, _ = R.attend(q.cpu(), k[blocks].cpu(), v[blocks].cpu(), c.k_scale[blocks].cpu(), c.v_scale[blocks].cpu(),
                           [[0, 1]], [200], [0, rows], float(np.float32(1 / np.sqrt(d))))
        assert rel(out, want) <= REL["f32"]
    c.check()


def test_step_in_a_cuda_graph(kv):
    """extend, append and attend of a decode step captured once and replayed with new contents."""
    c, *_ = cache_of(kv, "int8", 20, 2, 16, 64)
    tab, lens, free, nf = ints([[0, 1, 2, -1], [3, 4, -1, -1]]), ints([47, 20]), ints(list(range(19, 4, -1))), ints([15])
    new = ints([1, 1])
    x = torch.randn((2, 8, 64), device="cuda")

    def step():
        st = kv.extend_tables(tab, lens, new, free, nf, 2, 16)
        c.append(x[:, 4:6], x[:, 6:], st.slots)
        return c.attend(x[:, :4], tab, st.lens, st.cu, max_new=1)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(torch.randn((2, 8, 64), device="cuda"))
    g.replay()
    got = out.clone()
    assert torch.equal(got, step())


# ---- refusals ------------------------------------------------------------------------------------
def test_refusals(kv):
    E = kv.EngineError
    c, *_ = cache_of(kv, "int8", 4, 2, 16, 64)
    q = torch.randn((3, 4, 64), device="cuda")
    k = torch.randn((3, 2, 64), device="cuda")
    tab, lens, cu, slots = ints([[0, 1]]), ints([20]), ints([0, 3]), ints([0, 1, 2])
    from rusty_engine_b200._lib import RmoeError

    bad = [
        lambda: c.attend(q.cpu(), tab, lens, cu), lambda: c.attend(q.double(), tab, lens, cu),
        lambda: c.attend(q[..., :32], tab, lens, cu), lambda: c.attend(q.transpose(1, 2), tab, lens, cu),
        lambda: c.attend(q[:, :3], tab, lens, cu), lambda: c.attend(q, tab.long(), lens, cu),
        lambda: c.attend(q, tab[0], lens, cu), lambda: c.attend(q, tab, ints([1, 2]), cu),
        lambda: c.attend(q, tab, lens, ints([0])), lambda: c.attend(q, tab, lens, cu, window=-1),
        lambda: c.attend(q, tab, lens, cu, out=q.half()), lambda: c.attend(q, tab, lens, cu, out=q[:2]),
        lambda: c.append(k, k.half(), slots), lambda: c.append(k[:, :1], k, slots), lambda: c.append(k, k, slots[:2]),
        lambda: c.append(k, k, slots, q=q), lambda: c.append(k, k, slots, rope=kv.Rope(kv.RopeConfig(64), 8)),
        lambda: c.read(slots, torch.int32), lambda: c.read(slots.float()),
        lambda: kv.extend_tables(tab, lens, ints([1, 1]), ints([3]), ints([1]), 2, 16),
        lambda: kv.extend_tables(tab, lens, ints([1]), ints([3]), ints([1]), -1, 16),
        lambda: kv.extend_tables(tab.cpu(), lens, ints([1]), ints([3]), ints([1]), 1, 16),
        lambda: kv.Rope(kv.RopeConfig(63), 8), lambda: kv.Rope(kv.RopeConfig(64), 0),
        lambda: kv.Rope(kv.RopeConfig(64, scaling=kv.RopeScaling.Linear, factor=0.5), 8),
        lambda: kv.Rope(kv.RopeConfig(64, scaling=kv.RopeScaling.Yarn, factor=4.0), 8),
        lambda: kv.Rope(kv.RopeConfig(64, freq_factors=[1.0] * 31), 8),
        lambda: kv.Rope(kv.RopeConfig(64, freq_factors=[0.0] * 32), 8),
        lambda: kv.Rope(kv.RopeConfig(128), 8).apply(q, slots), lambda: kv.Rope(kv.RopeConfig(64), 8).apply(q, slots, k[:2]),
        lambda: kv.KVCache(0, 16, 1, 64), lambda: kv.KVCache.from_buffers(c.k, c.v, c.k_scale, c.v_scale[:2]),
        lambda: kv.KVCache.from_buffers(c.k.float(), c.v, c.k_scale, c.v_scale),
        lambda: kv.KVCache.from_buffers(c.k.transpose(0, 1), c.v.transpose(0, 1), c.k_scale.t(), c.v_scale.t()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(E):
            f()
            pytest.fail(f"case {i} was taken")
    for f in (lambda: kv.KVCache(2, 24, 1, 64), lambda: kv.KVCache(2, 16, 1, 96),
              lambda: kv.extend_tables(tab, lens, ints([1]), ints([3]), ints([1]), 1, 24),
              lambda: c.append(k, k, slots, rope=kv.Rope(kv.RopeConfig(24), 8), positions=slots)):
        with pytest.raises(RmoeError, match="UNSUPPORTED"):
            f()
    c.check()
