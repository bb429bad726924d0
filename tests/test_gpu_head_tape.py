"""The operators around a decoder's attention and loss as nodes of the tape (Rope, QkNormRope,
LinearCrossEntropy), and the decoder that uses them together: forward, tape backward, graph replay,
training steps.

Tolerances: a node's gradients are the direct call's, bit for bit; the decoder's are compared with fp32
torch autograd of the same bf16-stored forward at the 2e-2 of the other decoder tests (normwise: a
gradient passes some ten bf16 roundings of 2^-8 each, in sums that cancel)."""
import math

import numpy as np
import pytest

from conftest import rel_err

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


@pytest.fixture(scope="module")
def env(gpu):
    import gn_bwd
    import grilly_bridge as gb
    import grilly_core
    dev = grilly_core.Device(0)
    gb.attach_torch_stream(dev)
    return grilly_core, gb, dev, gn_bwd


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def rand(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def grad(gb, dev, tape, t, shape=None, dtype=None):
    gid = tape.get_grad_buffer(t.data_ptr())
    assert gid != 0, "no gradient recorded"
    return gb.download(dev, gid, t.shape if shape is None else shape, gb.dtype_code(t) if dtype is None else dtype)


def host(t):
    return t.float().cpu().numpy()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("with_positions", [False, True])
def test_rope_node(env, dtype, with_positions):
    gc, gb, dev, gn = env
    g = gen(1)
    B, S, H, D = 2, 9, 3, 64
    x, dy = rand(g, B, S, H * D, dtype=dtype), rand(g, B, S, H * D, dtype=dtype)
    f, m = gn.rope_freqs(32, scaling="yarn", factor=4.0)
    pos = torch.randint(0, 900, (B, S), device=DEV, generator=g).to(torch.int32) if with_positions else None
    kw = dict(mode="interleaved", mscale=m, positions=pos, pos0=0 if with_positions else 5)
    y = gn.rope_fwd(x.view(B, S, H, D), f, **kw)
    want = gn.rope_bwd(dy.view(B, S, H, D), f, **kw)
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(gc.OpType.Rope, [gb.tref(x, True)], [gb.tref(y.view(B, S, H * D))],
                       gb.rope_params(H, 32, "interleaved", m, with_positions, kw["pos0"]))
    tape.save_for_backward(n, [f.data_ptr(), pos.data_ptr() if with_positions else 0])
    tape.backward(n, dy.data_ptr())
    np.testing.assert_array_equal(grad(gb, dev, tape, x), host(want).reshape(B, S, H * D))
    tape.end()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("weights", [False, True])
def test_qk_norm_rope_node(env, dtype, weights):
    gc, gb, dev, gn = env
    g = gen(2)
    B, S, H, K, D = 2, 40, 4, 2, 64
    C = (H + 2 * K) * D
    x, dy = rand(g, B, S, C, dtype=dtype), rand(g, B, S, C, dtype=dtype)
    wq, wk = (rand(g, D, dtype=dtype), rand(g, D, dtype=dtype)) if weights else (None, None)
    f, _ = gn.rope_freqs(64)
    part = lambda t: (t.view(B, S, -1, D)[:, :, :H], t.view(B, S, -1, D)[:, :, H:H + K], t.view(B, S, -1, D)[:, :, H + K:])
    y, want = torch.empty_like(x), torch.empty_like(x)
    gn.qk_norm_rope_fwd(*part(x)[:2], wq, wk, f, v=part(x)[2], out=part(y), pos0=3, eps=1e-5)
    got = gn.qk_norm_rope_bwd(*part(dy)[:2], *part(x)[:2], wq, wk, f, dyv=part(dy)[2], out=part(want), pos0=3, eps=1e-5)
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(gc.OpType.QkNormRope, [gb.tref(x, True)], [gb.tref(y)],
                       gb.qk_norm_rope_params(H, K, 64, eps=1e-5, pos0=3))
    tape.save_for_backward(n, [wq.data_ptr() if weights else 0, wk.data_ptr() if weights else 0, f.data_ptr()])
    tape.backward(n, dy.data_ptr())
    np.testing.assert_array_equal(grad(gb, dev, tape, x), host(want))
    if weights:
        np.testing.assert_array_equal(grad(gb, dev, tape, wq, dtype=gb.DTYPE_F32), host(got[3]))
        np.testing.assert_array_equal(grad(gb, dev, tape, wk, dtype=gb.DTYPE_F32), host(got[4]))
    tape.end()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("upstream", [False, True])
def test_linear_cross_entropy_node(env, dtype, upstream):
    """With a tied table: the Embedding's gradient joins E's."""
    gc, gb, dev, gn = env
    g = gen(3)
    T, d, V = 50, 64, 300
    E = rand(g, V, d, dtype=dtype, std=0.3)
    ids = torch.randperm(V, device=DEV, generator=g)[:T].to(torch.int32)  # no id twice: no order to differ in
    h = E[ids.long()].contiguous()
    t = torch.randint(0, V, (T,), device=DEV, generator=g).to(torch.int32)
    t[::7] = -100
    u = torch.rand(T, device=DEV, generator=g)
    loss, lse = gn.linear_xent_fwd(h, E, t)
    dh, dE = gn.linear_xent_bwd(h, E, t, lse, dloss=u if upstream else None, scale=0.25)
    tape = gb.create_tape_context(dev)
    tape.begin()
    n = tape.record_op(gc.OpType.Embedding, [gb.tref(ids)], [gb.tref(h)], gb.embedding_params(V))
    tape.save_for_backward(n, [E.data_ptr()])
    n = tape.record_op(gc.OpType.LinearCrossEntropy, [gb.tref(h, True), gb.tref(t)], [gb.tref(loss)],
                       gb.linear_cross_entropy_params(V, 0.25))
    tape.save_for_backward(n, [E.data_ptr(), lse.data_ptr()])
    tape.backward(n, u.data_ptr() if upstream else 0)
    np.testing.assert_array_equal(grad(gb, dev, tape, h), host(dh))
    dE = dE.index_add(0, ids.long(), dh.float())
    np.testing.assert_array_equal(grad(gb, dev, tape, E, dtype=gb.DTYPE_F32), host(dE))
    tape.end()


def test_node_refusals(env):
    gc, gb, dev, gn = env
    x = torch.zeros(2, 4, 256, device=DEV, dtype=BF)
    y = torch.zeros_like(x)
    f, _ = gn.rope_freqs(64)
    t = torch.zeros(8, device=DEV, dtype=torch.int32)
    loss = torch.zeros(8, device=DEV)

    def go(op, ins, outs, params, saved, match, exc=ValueError):
        tape = gb.create_tape_context(dev)
        tape.begin()
        n = tape.record_op(op, ins, outs, params)
        tape.save_for_backward(n, saved)
        with pytest.raises(exc, match=match):
            tape.backward(n, y.data_ptr())
        tape.end()

    op, r = gc.OpType, gb.tref
    go(op.Rope, [r(x, True)], [r(y)], gb.rope_params(3, 64), [f.data_ptr()], "heads")
    go(op.Rope, [r(x, True)], [r(y)], gb.rope_params(4, 64), [0], "frequencies")
    go(op.Rope, [r(x, True)], [r(y)], gb.rope_params(4, 66), [f.data_ptr()], "rot", RuntimeError)
    go(op.QkNormRope, [r(x, True)], [r(y)], gb.qk_norm_rope_params(3, 1, 64), [0, 0, f.data_ptr()], "heads")
    go(op.QkNormRope, [r(x, True)], [r(x)], gb.qk_norm_rope_params(2, 1, 64), [0, 0, f.data_ptr()], "in its place")
    h = x.view(8, 256)
    go(op.LinearCrossEntropy, [r(h, True), r(t)], [r(loss)], b"", [x.data_ptr(), loss.data_ptr()], "vocabulary")
    go(op.LinearCrossEntropy, [r(h, True), r(t)], [r(loss)], gb.linear_cross_entropy_params(8), [x.data_ptr()], "lse")
    go(op.LinearCrossEntropy, [r(h, True), r(t[:4].contiguous())], [r(loss)], gb.linear_cross_entropy_params(8),
       [x.data_ptr(), loss.data_ptr()], "target")


def reference(m):
    """fp32 torch autograd of the decoder with both options, rounding to bf16 where the GPU run
    stores (straight through)."""
    rb = lambda t: t + (t.bfloat16().float() - t).detach()
    leaf = lambda t: t.detach().float().clone().requires_grad_(True)
    B, S, H, d, T = m.B, m.S, m.H, m.d, m.T
    D = d // H
    E = leaf(m.E)
    params = [{k: leaf(v) for k, v in p.items()} for p in m.layers]
    lnf_g, lnf_b = leaf(m.lnf_g), leaf(m.lnf_b)

    def ln(x, g, b):
        mu = x.mean(-1, keepdim=True)
        return rb((x - mu) * torch.rsqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5) * g + b)

    a = (torch.arange(S, device=DEV).double()[:, None] * m.freqs).float()
    cos, sin = torch.cos(a)[None, :, None], torch.sin(a)[None, :, None]

    def norm_rope(x, w):
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        u, v = n.chunk(2, -1)
        return rb(torch.cat((u * cos - v * sin, v * cos + u * sin), -1))

    def gelu(u):
        return 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3)))

    mask = torch.triu(torch.ones(S, S, dtype=torch.bool, device=DEV), 1)
    x = E[m.ids.long()]
    for p in params:
        qkv = rb(ln(x, p["ln1_g"], p["ln1_b"]) @ p["Wqkv"].t() + p["bqkv"]).view(B, S, 3, H, D)
        q, k, v = (t.permute(0, 2, 1, 3) for t in (norm_rope(qkv[:, :, 0], p["qn"]), norm_rope(qkv[:, :, 1], p["kn"]),
                                                   qkv[:, :, 2]))
        sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
        o = torch.matmul(torch.softmax(sc.masked_fill(mask, float("-inf")), -1), v)
        x2 = x + rb(rb(o.permute(0, 2, 1, 3).reshape(T, d)) @ p["Wo"].t() + p["bo"])
        n2 = ln(x2, p["ln2_g"], p["ln2_b"])
        h = rb(rb(n2 @ p["Wg"].t() + p["bg"]) * gelu(rb(n2 @ p["Wu"].t() + p["bu"])))
        x = x2 + rb(h @ p["Wd"].t() + p["bd"])
    logits = ln(x, lnf_g, lnf_b) @ E.t()
    torch.nn.functional.cross_entropy(logits, m.tgt.long()).backward()
    return E, params, lnf_g


def model(seed):
    import decoder_tape
    m = decoder_tape.Decoder(layers=2, d=128, heads=2, ff=256, vocab=301, batch=2, seq=129, seed=seed, qk_norm_rope=True,
                             fused_loss=True)
    g = gen(seed)
    for p in m.layers:
        for k in ("ln1_g", "ln2_g", "qn", "kn"):
            p[k].copy_((1 + 0.2 * torch.randn(p[k].shape, device=DEV, generator=g)).bfloat16())
        for k in ("ln1_b", "ln2_b", "bqkv", "bo", "bg", "bu", "bd"):
            p[k].copy_((0.05 * torch.randn(p[k].shape, device=DEV, generator=g)).bfloat16())
    return m


KEYS = ("Wqkv", "bqkv", "Wo", "ln1_g", "ln2_b", "Wg", "Wu", "bu", "Wd", "qn", "kn")


def test_decoder_with_both_options(env):
    gc, gb, dev, gn = env
    m = model(7)
    m.forward()
    tape = gb.create_tape_context(dev)
    tape.begin()
    tape.backward(m.record(tape), 0)
    got = {"E": grad(gb, dev, tape, m.E, dtype=gb.DTYPE_F32), "lnf_g": grad(gb, dev, tape, m.lnf_g, dtype=gb.DTYPE_F32)}
    for i, p in enumerate(m.layers):
        got.update({f"{k}{i}": grad(gb, dev, tape, p[k], dtype=gb.DTYPE_F32) for k in KEYS})
    tape.end()
    E, params, lnf_g = reference(m)
    want = {"E": E.grad, "lnf_g": lnf_g.grad}
    for i, p in enumerate(params):
        want.update({f"{k}{i}": p[k].grad for k in KEYS})
    errs = {k: rel_err(got[k], want[k].cpu().numpy()) for k in got}
    bad = {k: v for k, v in errs.items() if not v < 2e-2}
    assert not bad, f"relative errors above 2e-2: {bad} (all: {errs})"


def test_decoder_backward_replayed(env):
    """Captured once into a graph of kernel nodes only; replays with changed targets equal the eager
    backward (the tied table, whose embedding part sums fp32 atomics, within 1e-6)."""
    gc, gb, dev, gn = env
    m = model(8)
    m.forward()
    tensors = {"E": m.E, "lnf_g": m.lnf_g}
    for i, p in enumerate(m.layers):
        tensors.update({f"{k}{i}": p[k] for k in KEYS})
    tape = gb.create_tape_context(dev)
    tape.begin()
    graph = gc.OpGraph()
    graph.capture_backward(tape, m.record(tape), 0)
    tape.end()
    assert graph.node_counts()["memset"] == 0 and graph.node_counts()["memcpy"] == 0
    g = gen(9)
    for rep in range(3):
        if rep:
            m.tgt.copy_(torch.randint(0, m.V, m.tgt.shape, device=DEV, generator=g, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.execute(dev)
        torch.cuda.synchronize()
        eager = gb.create_tape_context(dev)
        eager.begin()
        eager.backward(m.record(eager), 0)
        for k, t in tensors.items():
            a = gb.download(dev, graph.get_grad_buffer(t.data_ptr()), t.shape, gb.DTYPE_F32)
            b = grad(gb, dev, eager, t, dtype=gb.DTYPE_F32)
            if k == "E":
                assert rel_err(a, b) < 1e-6
            else:
                np.testing.assert_array_equal(a, b, err_msg=f"replay {rep}: {k}")
        eager.end()
    graph.clear()


def test_training_steps(env):
    """Three steps of forward, tape backward and AdamW: every weight with a gradient moves, and stays
    finite."""
    gc, gb, dev, gn = env
    m = model(10)
    weights = [m.E, m.lnf_g] + [p[k] for p in m.layers for k in KEYS]
    before = [w.clone() for w in weights]
    opt = gb.AdamW(weights, lr=1e-2)
    tape = gb.create_tape_context(dev)
    for _ in range(3):
        m.forward()
        tape.begin()
        tape.backward(m.record(tape), 0)
        assert opt.step(tape) == len(weights)
        tape.end()
    torch.cuda.synchronize()
    for w, b in zip(weights, before):
        assert bool(torch.isfinite(w).all()) and not torch.equal(w, b)
