"""A decoder stack driven through the tape engine: the end-to-end backward workload.

Per layer (pre-LN):  n1 = LN(x);  qkv = n1 Wqkv^T + bqkv;  o = causal attention over the
fused qkv rows;  x2 = x + o Wo^T + bo;  n2 = LN(x2);  h = gate * GELU_tanh(up) with
gate = n2 Wg^T + bg, up = n2 Wu^T + bu;  x3 = x2 + h Wd^T + bd.
Embedding x0 = E[ids], final LN, tied LM head logits = LN(x_L) E^T, cross-entropy over the
vocabulary (scale 1/T).  bf16 weights and block activations, fp32 statistics and weight
gradients; the residual stream x (and so its gradient) is fp32: the norms read it in fp32 and
write bf16, each bf16 branch output is added into it in fp32.  Carried in bf16, the residual
gradient's rounding over the 12 layers reaches the LayerNorm gains' gradient (a sum that
cancels heavily) at a few percent; in fp32 it stays within the bf16 tolerance.

Two options replace parts of it: `qk_norm_rope` norms queries and keys per head (weights qn, kn
[D]) and rotates them by position between the projection and the attention (gn_qk_norm_rope_fwd);
`fused_loss` takes the loss from the last norm's output and E (gn_linear_xent_fwd): no logits and no
gradient of them are kept.

Three more say how a block ends: `residual_norm` takes the residual sum and the next norm in one pass
(gn_residual_norm_fwd), with `dropout` on each branch in it and on the embedding (gn_dropout_fwd; masks from `seed`, the
place and the step counter `self.step`, an int64 on the GPU); `fused_linear` adds the products that end a branch into
the stream in their epilogue (gn_linear_act_fwd); `ffn="gelu"` has a feed-forward of two products, the first with its
activation in the epilogue.

`Decoder.forward()` runs the forward on the GPU through this library's forward kernels
(untimed: gn_layernorm_fwd saving mean/rstd, gn_linear_fwd, gn_glu_linear_fwd saving the
gate/up caches, gn_attn_fwd saving the fp32 row logsumexp; torch only for the embedding
gather and the residual adds) and keeps every tensor the backward needs.  `Decoder.record(tape)`
records the nodes the reference's tape would hold for this model (Linear, LayerNorm,
FlashAttention2, Add, CrossEntropy; autograd.h:81-141) plus this build's FusedGLU and
Embedding nodes, with the saved-slot conventions of each handler.
"""
import torch

import grilly_bridge as gb
import grilly_core
import gn_bwd as gn


class Decoder:
    def __init__(self, layers=12, d=768, heads=12, ff=3072, vocab=32000, batch=8, seq=1024,
                 seed=5, device="cuda:0", glu_epilogue=True, qk_norm_rope=False, fused_loss=False,
                 residual_norm=False, dropout=0.0, fused_linear=False, ffn="geglu"):
        if dropout and not residual_norm:
            raise ValueError("dropout goes with residual_norm")
        if fused_linear and residual_norm:
            raise ValueError("residual_norm and fused_linear each take the residual sum")
        if ffn not in ("geglu", "gelu"):
            raise ValueError(f"ffn {ffn!r}: geglu or gelu")
        self.residual_norm, self.p, self.fused_linear, self.ffn, self.seed = residual_norm, dropout, fused_linear, ffn, seed
        self.L, self.d, self.H, self.ff, self.V = layers, d, heads, ff, vocab
        self.glu_epilogue, self.qk_norm_rope, self.fused_loss = glu_epilogue, qk_norm_rope, fused_loss
        self.B, self.S, self.T = batch, seq, batch * seq
        self.dev = torch.device(device)
        g = torch.Generator(device=self.dev)
        g.manual_seed(seed)
        bf = torch.bfloat16

        def w(*shape):
            return (torch.randn(*shape, device=self.dev, generator=g) * 0.02).to(bf).contiguous()

        def const(n, v):
            return torch.full((n,), float(v), device=self.dev, dtype=bf)

        self.E = w(vocab, d)
        self.layers = [dict(ln1_g=const(d, 1), ln1_b=const(d, 0), Wqkv=w(3 * d, d),
                            bqkv=const(3 * d, 0), Wo=w(d, d), bo=const(d, 0), ln2_g=const(d, 1),
                            ln2_b=const(d, 0), Wg=w(ff, d), Wu=w(ff, d), bg=const(ff, 0),
                            bu=const(ff, 0), Wd=w(d, ff), bd=const(d, 0))
                       for _ in range(layers)]
        if qk_norm_rope:
            for p in self.layers:
                p["qn"], p["kn"] = const(d // heads, 1), const(d // heads, 1)
            self.freqs, self.mscale = gn.rope_freqs(d // heads, device=self.dev)
        self.lnf_g, self.lnf_b = const(d, 1), const(d, 0)
        self.step = torch.zeros(1, device=self.dev, dtype=torch.int64)
        ids = torch.randint(0, vocab, (batch, seq), device=self.dev, generator=g)
        self.ids = ids.reshape(-1).to(torch.int32).contiguous()
        self.tgt = torch.roll(ids, -1, dims=1).reshape(-1).to(torch.int32).contiguous()
        self.loss = torch.zeros(1, device=self.dev)
        self.acts = None

    # ------------------------------------------------------------------ forward (untimed)
    def forward(self):
        B, S, H, d, T = self.B, self.S, self.H, self.d, self.T
        D = d // H
        ws = gn.workspace(gn.attn_workspace_bytes(B, H, S, D, gn.BF16), self.dev)
        bf = torch.bfloat16
        x = self.E[self.ids.long()].float().contiguous()  # fp32 residual stream
        self.x0 = x
        if self.p:
            x = self.x0d = gn.dropout_fwd(x, self.p, self.seed, stream=0, step=self.step)
        acts = []
        n1 = None
        for i, p in enumerate(self.layers):
            a = {"x": x}
            if n1 is None:
                a["n1"], a["m1"], a["r1"] = gn.layernorm_fwd(x, p["ln1_g"], p["ln1_b"], out_dtype=bf)
            else:
                a["n1"] = n1
            a["qkv"] = gn.linear_fwd(a["n1"], p["Wqkv"], p["bqkv"])
            if self.qk_norm_rope:
                # the rows the attention's backward reads, and from them the forward's heads
                a["rot"] = torch.empty_like(a["qkv"])
                parts = [[t.view(B, S, 3, H, D)[:, :, i] for i in range(3)] for t in (a["qkv"], a["rot"])]
                gn.qk_norm_rope_fwd(*parts[0][:2], p["qn"], p["kn"], self.freqs, v=parts[0][2], mscale=self.mscale,
                                    out=parts[1])
            rows = a["rot"] if self.qk_norm_rope else a["qkv"]
            q, k, v = (t.contiguous() for t in rows.view(B, S, 3, H, D).permute(2, 0, 3, 1, 4))
            O, a["lse"] = gn.attn_fwd(q, k, v, causal=True, rope="none", ws=ws)
            a["o"] = O.permute(0, 2, 1, 3).reshape(T, d).contiguous()
            if self.fused_linear:
                a["x2"] = gn.linear_act_fwd(a["o"], p["Wo"], p["bo"], residual=x)
            else:
                a["ao"] = gn.linear_fwd(a["o"], p["Wo"], p["bo"])
            if self.residual_norm:
                a["x2"], a["n2"] = self._branch(a["ao"], x, p["ln2_g"], p["ln2_b"], 2 * i + 1)
            else:
                if not self.fused_linear:
                    a["x2"] = (x + a["ao"].float()).contiguous()
                a["n2"], a["m2"], a["r2"] = gn.layernorm_fwd(a["x2"], p["ln2_g"], p["ln2_b"], out_dtype=bf)
            if self.ffn == "gelu":
                a["h"], a["pre"] = gn.linear_act_fwd(a["n2"], p["Wu"], p["bu"], act="gelu_tanh", need_pre=True)
            else:
                a["gate"], a["up"], a["h"] = gn.glu_linear_fwd("geglu_up", a["n2"], p["Wg"], p["Wu"],
                                                               p["bg"], p["bu"])
            if self.fused_linear:
                a["x3"] = gn.linear_act_fwd(a["h"], p["Wd"], p["bd"], residual=a["x2"])
            else:
                a["f"] = gn.linear_fwd(a["h"], p["Wd"], p["bd"])
            if self.residual_norm:
                a["x3"], n1 = self._branch(a["f"], a["x2"], *self._norm_after(i), 2 * i + 2)
            elif not self.fused_linear:
                a["x3"] = (a["x2"] + a["f"].float()).contiguous()
            acts.append(a)
            x = a["x3"]
        if self.residual_norm:
            self.nf = n1
        else:
            self.nf, self.mf, self.rf = gn.layernorm_fwd(x, self.lnf_g, self.lnf_b, out_dtype=bf)
        if self.fused_loss:
            self.row_loss, self.lse = gn.linear_xent_fwd(self.nf, self.E, self.tgt)
        else:
            self.logits = gn.linear_fwd(self.nf, self.E)
        self.acts = acts
        torch.cuda.synchronize()

    def _norm_after(self, i):
        """The weights of the norm behind layer i: the next layer's first, or the last one."""
        if i + 1 < self.L:
            return self.layers[i + 1]["ln1_g"], self.layers[i + 1]["ln1_b"]
        return self.lnf_g, self.lnf_b

    def _branch(self, h, x, w, b, place):
        return gn.residual_norm_fwd(h, x, pre="layer", pre_w=w, pre_b=b, p=self.p, seed=self.seed, stream=place, step=self.step)

    # ------------------------------------------------------------------ tape
    def record(self, tape):
        """Record the forward's nodes (the forward must have run); returns the loss node."""
        assert self.acts is not None, "run forward() first"
        op, t, P = grilly_core.OpType, gb.tref, (lambda x: x.data_ptr())
        B, S, H, d = self.B, self.S, self.H, self.d
        n = tape.record_op(op.Embedding, [t(self.ids)], [t(self.x0)], gb.embedding_params(self.V))
        tape.save_for_backward(n, [P(self.E)])
        if self.p:
            n = tape.record_op(op.Dropout, [t(self.x0, True)], [t(self.x0d)], gb.dropout_params(self.p, self.seed))
            tape.save_for_backward(n, [P(self.step)])

        def branch(h, x, y, z, w, b, place):
            n = tape.record_op(op.ResidualNorm, [t(h, True), t(x, True)], [t(y), t(z)],
                               gb.residual_norm_params(pre="layer", p=self.p, seed=self.seed, stream=place))
            tape.save_for_backward(n, [0, 0, P(w), P(b), 0, P(self.step)])

        for i, (p, a) in enumerate(zip(self.layers, self.acts)):
            if "m1" in a:
                n = tape.record_op(op.LayerNorm, [t(a["x"], True)], [t(a["n1"])], gb.layernorm_params())
                tape.save_for_backward(n, [P(p["ln1_g"]), P(p["ln1_b"]), P(a["m1"]), P(a["r1"])])
            n = tape.record_op(op.Linear, [t(a["n1"], True)], [t(a["qkv"])])
            tape.save_for_backward(n, [P(p["Wqkv"]), P(p["bqkv"])])
            rows = a["qkv"]
            if self.qk_norm_rope:
                D = d // H
                rows = a["rot"]
                n = tape.record_op(op.QkNormRope, [gb.make_tensor_ref(P(a["qkv"]), (B, S, 3 * d), gb.DTYPE_BF16, True)],
                                   [gb.make_tensor_ref(P(rows), (B, S, 3 * d), gb.DTYPE_BF16)],
                                   gb.qk_norm_rope_params(H, H, D, mscale=self.mscale))
                tape.save_for_backward(n, [P(p["qn"]), P(p["kn"]), P(self.freqs)])
            qkv = gb.make_tensor_ref(P(rows), (B, S, 3 * d), gb.DTYPE_BF16, True)
            o = gb.make_tensor_ref(P(a["o"]), (B, S, d), gb.DTYPE_BF16)
            n = tape.record_op(op.FlashAttention2, [qkv], [o],
                               gb.attention_params(causal=True, rope="none", fused_qkv_heads=H))
            tape.save_for_backward(n, [P(a["lse"])])
            def ends_branch(x, W, b, out, stream, y):
                """The product that ends a branch, and the residual sum."""
                if self.fused_linear:
                    n = tape.record_op(op.LinearAct, [t(x, True), t(stream, True)], [t(y)], gb.linear_act_params())
                else:
                    n = tape.record_op(op.Linear, [t(x, True)], [t(out)])
                tape.save_for_backward(n, [P(W), P(b)])
                if not self.fused_linear and not self.residual_norm:
                    tape.record_op(op.Add, [t(stream, True), t(out, True)], [t(y)])

            ends_branch(a["o"], p["Wo"], p["bo"], a.get("ao"), a["x"], a["x2"])
            if self.residual_norm:
                branch(a["ao"], a["x"], a["x2"], a["n2"], p["ln2_g"], p["ln2_b"], 2 * i + 1)
            else:
                n = tape.record_op(op.LayerNorm, [t(a["x2"], True)], [t(a["n2"])], gb.layernorm_params())
                tape.save_for_backward(n, [P(p["ln2_g"]), P(p["ln2_b"]), P(a["m2"]), P(a["r2"])])
            if self.ffn == "gelu":
                n = tape.record_op(op.LinearAct, [t(a["n2"], True)], [t(a["h"])], gb.linear_act_params("gelu_tanh"))
                tape.save_for_backward(n, [P(p["Wu"]), P(p["bu"]), P(a["pre"])])
            else:
                n = tape.record_op(op.FusedGLU, [t(a["n2"], True)], [t(a["h"])],
                                   gb.fused_glu_params("geglu_up"))
                tape.save_for_backward(n, [P(p["Wg"]), P(p["Wu"]), P(a["gate"]), P(a["up"]),
                                           P(p["bg"]), P(p["bu"])])
            ends_branch(a["h"], p["Wd"], p["bd"], a.get("f"), a["x2"], a["x3"])
            if self.residual_norm:
                z = self.acts[i + 1]["n1"] if i + 1 < self.L else self.nf
                branch(a["f"], a["x2"], a["x3"], z, *self._norm_after(i), 2 * i + 2)
        last = self.acts[-1]["x3"]
        if not self.residual_norm:
            n = tape.record_op(op.LayerNorm, [t(last, True)], [t(self.nf)], gb.layernorm_params())
            tape.save_for_backward(n, [P(self.lnf_g), P(self.lnf_b), P(self.mf), P(self.rf)])
        if self.fused_loss:
            n = tape.record_op(op.LinearCrossEntropy, [t(self.nf, True), t(self.tgt)], [t(self.row_loss)],
                               gb.linear_cross_entropy_params(self.V, 1.0 / self.T))
            tape.save_for_backward(n, [P(self.E), P(self.lse)])
            return n
        n = tape.record_op(op.Linear, [t(self.nf, True)], [t(self.logits)])
        tape.save_for_backward(n, [P(self.E)])
        return tape.record_op(op.CrossEntropy, [t(self.logits, True), t(self.tgt)], [t(self.loss)],
                              gb.cross_entropy_params(1.0 / self.T))

    def backward_step(self, tape):
        """One end-to-end backward through the tape: begin, record, backward, end.  The tape
        runs with set_glu_epilogue(True): each down projection forms its GLU's local gradients
        in its input-gradient GEMM (the GLU output's gradient is not kept)."""
        tape.set_glu_epilogue(self.glu_epilogue)
        tape.begin()
        loss = self.record(tape)
        tape.backward(loss, 0)
        tape.end()

    def flops(self):
        """Backward GEMM + attention FLOPs (dX and dW of every projection, causal attention
        with the P recompute counted once: 5 products over half the score matrix)."""
        T, d, ff, V, S, H = self.T, self.d, self.ff, self.V, self.S, self.H
        up = 2 if self.ffn == "geglu" else 1
        per_layer = (2 * 2 * T * d * 3 * d + 2 * 2 * T * d * d + 2 * 2 * T * d * ff * up
                     + 2 * 2 * T * ff * d + 5 * 2.0 * S * S * (d // H) * 0.5 * self.B * H)
        return self.L * per_layer + 2 * 2 * T * d * V

    def fwd_flops(self):
        """Forward GEMM + attention FLOPs: every projection once, causal attention as 2
        products over half the score matrix, the LM head."""
        T, d, ff, V, S, H = self.T, self.d, self.ff, self.V, self.S, self.H
        up = 2 if self.ffn == "geglu" else 1
        per_layer = (2 * T * d * 3 * d + 2 * T * d * d + 2 * T * d * ff * up + 2 * T * ff * d
                     + 2 * 2.0 * S * S * (d // H) * 0.5 * self.B * H)
        return self.L * per_layer + 2 * T * d * V
