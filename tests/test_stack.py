"""The config-4 harness (rusty_engine_b200.stack): MoE transformer blocks around the layer,
against the CPU restatement of rusty-engine's prefill block with the MoE FFN
(oracle/stack_ref.py: src/forward.rs:532-571 with src/moe.rs:443-469), on a two-block stack of
small shapes, through both expert-product paths (40 tokens: decode kernels; 300 tokens:
tcgen05 kernels).  Hidden states after every block within relative L2 5e-3."""
import numpy as np
import pytest

from rusty_engine_b200 import synth


def small_geometry():
    from rusty_engine_b200.stack import Geometry

    return Geometry(d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, n_experts=8, top_k=2, inter=256,
                    rope_freq_base=1e6, rms_eps=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 300])
def test_stack_matches_reference_block(gpu, T):
    """Each part of each block against the CPU restatement on the GPU's own input to that part,
    so that the check is the part's error, not errors carried in from earlier parts: the
    attention residual y = x + o(attention(rmsnorm(x))) (the QMat products' fp16 operands) and
    the MoE FFN on rmsnorm(y) (the layer contract); relative L2 <= 5e-3 each."""
    import torch

    from oracle import stack_ref
    from rusty_engine_b200.stack import MoEStack, make_block, rope_tables

    g = small_geometry()
    blocks = [make_block(g, seed=10 + i, dlo=0.001, dhi=0.004, attn_dlo=0.002, attn_dhi=0.01) for i in range(2)]
    x = synth.activations(T, g.d_model, seed=T)
    stack = MoEStack(g, blocks, device=0)
    out = stack.forward(torch.from_numpy(x).cuda(), collect=True).cpu().numpy()
    ins = [t.cpu().numpy() for t in stack.block_inputs]
    mids = [t.cpu().numpy() for t in stack.block_mids]
    assert len(stack.moe_ms) == 2 and all(ms > 0 for ms in stack.moe_ms)
    stack.close()
    assert np.isfinite(out).all()
    cos, sin = rope_tables(g, T)
    outs = ins[1:] + [out]
    rel = lambda a, b: float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b))
    for i, b in enumerate(blocks):
        ra = rel(mids[i], stack_ref.attention_residual(g, b, ins[i], cos, sin))
        rm = rel(outs[i] - mids[i], stack_ref.moe_residual(g, b, mids[i]))
        print(f"stack T={T} block {i}: attention residual rel-L2 {ra:.2e}, MoE FFN rel-L2 {rm:.2e}")
        assert ra <= 5e-3 and rm <= 5e-3, (i, ra, rm)


def test_rope_tables_match_reference_formula():
    """cos / sin of pos * base^(-2i/d) in f32 (src/infer.rs:90-96, 115-127)."""
    from rusty_engine_b200.stack import rope_tables

    g = small_geometry()
    c, s = rope_tables(g, 5, pos_start=3)
    d = g.head_dim
    for pos in (3, 7):
        for i in (0, 1, 63):
            f = np.float32(1.0) / np.power(np.float32(g.rope_freq_base), np.float32(2 * i) / np.float32(d))
            ang = np.float32(pos) * np.float32(f)
            assert c[pos - 3, i] == np.float32(np.cos(ang)) and s[pos - 3, i] == np.float32(np.sin(ang))


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["Int8", "E4M3"])
def test_stack_serving_steps(gpu, code):
    """MoEStack.step over prompts, chunks and single tokens of three requests: every block's
    attention residual against a float64 restatement over the keys and values that the cache holds
    (relative L2 <= 5e-3, the bar of the prefill test: the QMat products' fp16 operands), and those
    values against the exact rotated keys and values, off by at most a rounding step of the cache
    (half a step, and half again for each time a block's scale grew)."""
    import torch

    from oracle import stack_ref
    from rusty_engine_b200 import kv
    from rusty_engine_b200.stack import MoEStack, make_block, rope_tables

    g = small_geometry()
    blocks = [make_block(g, seed=30 + i, dlo=0.001, dhi=0.004, attn_dlo=0.002, attn_dhi=0.01) for i in range(2)]
    stack = MoEStack(g, blocks, device=0)
    stack.open_cache(max_requests=3, n_blocks=40, block_size=16, max_pos=512, code=kv.CacheCode[code])
    steps = [[33, 0, 150], [1, 20, 1], [17, 1, 0], [1, 1, 1]]
    xs, ins, mids, outs = [], [[] for _ in blocks], [[] for _ in blocks], []
    req, pos, lens = [], [], [0, 0, 0]
    for i, new in enumerate(steps):
        x = synth.activations(sum(new), g.d_model, seed=50 + i)
        xs.append(x)
        outs.append(stack.step(torch.from_numpy(x).cuda(), torch.tensor(new, dtype=torch.int32, device="cuda"),
                               max_new=max(new), collect=True).cpu().numpy())
        for b in range(len(blocks)):
            ins[b].append(stack.block_inputs[b].cpu().numpy())
            mids[b].append(stack.block_mids[b].cpu().numpy())
        for r, n in enumerate(new):
            req += [r] * n
            pos += range(lens[r], lens[r] + n)
            lens[r] += n
    req, pos = np.array(req), np.array(pos)
    assert stack.batch.lens.tolist() == lens
    table = stack.batch.table.cpu().numpy()
    cos, sin = rope_tables(g, 512)
    hd, qd, kvd = g.head_dim, g.n_heads * g.head_dim, g.n_kv_heads * g.head_dim
    rel = lambda a, b: float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b))
    for b, w in enumerate(blocks):
        x = np.concatenate(ins[b])
        xn = stack_ref.rmsnorm(x, w.attn_norm, g.rms_eps)
        q = stack_ref.rope(stack_ref.proj(w.q, qd, g.d_model, xn), g.n_heads, hd, cos[pos], sin[pos])
        k = stack_ref.rope(stack_ref.proj(w.k, kvd, g.d_model, xn), g.n_kv_heads, hd, cos[pos], sin[pos])
        v = stack_ref.proj(w.v, kvd, g.d_model, xn)
        slots = torch.tensor(table[req, pos // 16] * 16 + pos % 16, dtype=torch.int32, device="cuda")
        ck, cv = (t.cpu().numpy().reshape(-1, kvd) for t in stack.caches[b].read(slots))
        stack.caches[b].check()
        # a step is max|x| / 127 of the block and head (1 / 16 of the value itself for e4m3, whose
        # last bit is a half of an eighth); the products' own error is 5e-3 of the row's size
        for got, want in ((ck, k), (cv, v)):
            unit = 3 / 127 if code == "Int8" else 3 / 16
            assert np.abs(got - want).max() <= unit * np.abs(want).max()
        ctx = np.zeros((len(req), qd))
        for t in range(len(req)):
            seen = (req == req[t]) & (pos <= pos[t])
            for h in range(g.n_heads):
                c = slice(h // (g.n_heads // g.n_kv_heads) * hd, (h // (g.n_heads // g.n_kv_heads) + 1) * hd)
                z = ck[seen][:, c].astype(np.float64) @ q[t, h * hd:(h + 1) * hd] / np.sqrt(hd)
                p = np.exp(z - z.max())
                ctx[t, h * hd:(h + 1) * hd] = p @ cv[seen][:, c].astype(np.float64) / p.sum()
        want = x + stack_ref.proj(w.o, g.d_model, qd, ctx)
        # attention before a block's scale grew saw codes of the smaller step: the cache's rounding
        e = rel(np.concatenate(mids[b]), want)
        print(f"stack step {code} block {b}: attention residual rel-L2 {e:.2e}")
        assert e <= (5e-3 if code == "Int8" else 2e-2)
    stack.finish(torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda"))
    assert stack.batch.lens.tolist() == [0, lens[1], 0]
    stack.close()
