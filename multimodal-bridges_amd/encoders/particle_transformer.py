"""MultiModalParticleTransformer on the HIP path (reference: encoders/particle_transformer.py:8-167).

Same constructor (config), module tree and parameter names as the reference -- the encoder layers ARE
torch's nn.TransformerEncoderLayer objects, kept as parameter containers only (so `transformer.layers.{i}.
self_attn.in_proj_weight`, `.linear1.weight`, `.norm1.weight` ... load from a reference checkpoint); their
forward is never called.  What runs instead, per TransformerEncoderBlock:

  h = input_proj(x) + time_proj(t * mask)      ONE mmb_linear_cat over [x rows | per-jet time embedding x mask]
  per layer (post-LN, ReLU FFN, as built at particle_transformer.py:29-35):
      qkv = in_proj(h)                         mmb_linear_cat
      a   = attention(qkv)                     mmb_attention_fwd -- keys restricted to the slots with mask == 0:
                                               the reference passes src_key_padding_mask = mask > 0 (:50, quirk Q4),
                                               so every slot attends to the PADDED slots only; a jet without a
                                               padded slot gets zeros (torch's safe softmax), i.e. out_proj.bias
      h   = LayerNorm1(h + out_proj(a))        mmb_linear_cat (+ residual epilogue), mmb_layernorm_fwd
      h   = LayerNorm2(h + linear2(relu(linear1(h))))

Deviation (documented in DESIGN.md): under torch.no_grad() + eval() the reference runs torch's fused / nested-tensor
inference kernels, which return NaN for a jet without a padded slot and zeros for the real particles when every
jet's padded slots come first; this implementation always follows the training-path arithmetic (identical
everywhere else: the goldens' generation runs agree).

Dropout (training mode, encoder.dropout > 0) sits where nn.TransformerEncoderLayer has it: on the attention
probabilities (mmb_attention_dropout_fwd), after out_proj (dropout1), after the FFN's ReLU, after linear2 (dropout2);
Philox masks keyed by (model seed, per-call offset), regenerated by the reverse pass.  Same law as torch's, another
random stream: checked statistically and, with the masks extracted, exactly (tests/test_hip_transformer.py).

encoder.checkpoint_bits: 8 keeps the activations of the layers in 8 bits between forward and reverse pass (checkpoint8.py):
a quarter of the tape; the attention runs once more in the reverse pass, on the decoded rows.
"""
import os
from types import SimpleNamespace

import torch
from torch import nn

from tensorclass import TensorMultiModal
from encoders.epic import WNLinear, ExecCtx, TimeSeg, _time_seg
from encoders.embedder import LocalState
from encoders.multimodal_epic import _unpack, _Head
from mmb_hip import ops
from mmb_hip import fused as fused_epic
from mmb_hip.ops import SEG_ROW
from encoders.checkpoint8 import Keep8, activations


class PlainLinear:
    """cat_s[X_s] @ cat_s[W_s]^T + sum_s b_s for plain (not weight-normed) nn.Linear parameters; a part with
    weight None is an identity (the reference's `time_proj = nn.Identity()` when d_time == d_model)."""

    def __init__(self, dim_out, parts, biases):
        self.dim_out = dim_out
        self.parts = parts              # [(weight Parameter (dim_out, k) | None, k)]
        self.biases = biases            # [bias Parameter (dim_out)]
        self.K = sum(k for _, k in parts)
        self._cache = None

    def weight(self):
        ws = [w for w, _ in self.parts if w is not None]
        key = tuple((w._version, w.data_ptr()) for w in ws) + tuple((b._version, b.data_ptr()) for b in self.biases)
        if self._cache is None or self._cache[0] != key:
            dev = self.biases[0].device
            if len(self.parts) == 1:
                W = self.parts[0][0].detach()
            else:
                W = torch.cat([w.detach() if w is not None else torch.eye(self.dim_out, k, device=dev)
                               for w, k in self.parts], dim=1).contiguous()
            b = self.biases[0].detach() if len(self.biases) == 1 else sum(b.detach() for b in self.biases)
            self._cache = (key, W, b.contiguous())
        return self._cache[1]

    def bias(self):
        self.weight()
        return self._cache[2]

    def run(self, ctx, segs, act=None, res1=None, out=None, norm=None, dropout=False):
        """y = act(cat(segs) @ W^T + b) + res1;  with norm (an nn.LayerNorm): LayerNorm(y), in the same call
        (mmb_linear_cat_ln: the post-LN sublayer of nn.TransformerEncoderLayer).
        dropout (and ctx.drop_p > 0): y = dropout(act(cat(segs) @ W^T + b)) + res1 -- the residual joins AFTER the
        dropout, x + dropout(sublayer(x)) -- through the two-stage epilogue of mmb_linear_cat (Philox mask keyed by the
        context's next offset, regenerated by mmb_act_bwd); the LayerNorm is then a launch of its own."""
        W = self.weight()
        p = ctx.drop_p if (dropout and ctx.drop_p > 0.0) else 0.0
        rec = ctx.recording
        if p > 0.0:
            off = ctx.next_offset()
            _, y2 = ops.linear_cat(segs, W, self.bias(), ctx.N, maskf=ctx.mi.maskf, act=act, res2=res1, want_y1=False,
                                   out2=out if (norm is None and out is not None) else
                                   torch.empty(segs[0][0].shape[0], self.dim_out, dtype=torch.float32, device=W.device),
                                   drop_p=p, seed=ctx.seed, offset=off)
            if rec:                                       # relu' comes from y2 itself (mmb_act_bwd): y1 is never stored
                ctx.tape.append(("plinear", self, ctx.N, segs, act, None, None, res1, None, None, y2, p, off))
            if norm is None:
                return y2
            r = ops.layernorm_fwd(y2, norm.weight.detach(), norm.bias.detach(), norm.eps, want_stats=rec, out=out)
            if rec:
                ctx.tape.append(("ln", y2, r[0], r[1], norm))
                return r[0]
            return r
        if norm is None:
            y = ops.linear_cat(segs, W, self.bias(), ctx.N, maskf=ctx.mi.maskf, act=act, residual=res1, out=out)
            if rec:
                ctx.tape.append(("plinear", self, ctx.N, segs, act, res1, None, None, None, y, None, 0.0, 0))
            return y
        y1, y, stats = ops.linear_cat_ln(segs, W, self.bias(), ctx.N, norm.weight.detach(), norm.bias.detach(), norm.eps,
                                         maskf=ctx.mi.maskf, act=act, residual=res1, want_y1=rec, want_stats=rec, out=out)
        if rec:                                           # the same two tape entries as the unfused pair
            ctx.tape.append(("plinear", self, ctx.N, segs, act, res1, None, None, None, y1, None, 0.0, 0))
            ctx.tape.append(("ln", y1, y, stats, norm))
        return y


class _JetRowAttention:
    """The attention of the compacted inference path: with uniform keys (quirk Q4 + masked inputs) the output of every
    query of a jet is the V row of the jet's padded slots -- a row gather.  `rows` (M',) int32: for each compact row the
    compact row of its jet's representative, -1 for a jet without padded slots (no valid key: zeros).  The fused layer
    tail gathers through `rows` itself; layered layers call the object."""

    def __init__(self, cp):
        self.cp, self.rows = cp, cp.src

    def __call__(self, qkv):
        d = qkv.shape[1] // 3
        v = qkv[:, 2 * d:].index_select(0, self.cp.src.clamp(min=0).long())
        return v if self.cp.all_pad else v * self.cp.has_pad.index_select(0, self.cp.jet)


class TransformerEncoderBlock(nn.Module):
    def __init__(self, d_input, d_model, d_time, n_layers, n_heads, dim_feedforward, dropout):
        super().__init__()
        self.input_proj = nn.Linear(d_input, d_model)
        self.time_proj = nn.Linear(d_time, d_model) if d_time != d_model else nn.Identity()
        layer = nn.TransformerEncoderLayer(d_model=d_model, nhead=n_heads, dim_feedforward=dim_feedforward,
                                           dropout=dropout, batch_first=True)
        self.transformer = nn.TransformerEncoder(layer, num_layers=n_layers, enable_nested_tensor=False)
        self.n_heads, self.d_model, self.d_time, self.p_drop = n_heads, d_model, d_time, dropout
        self._specs = None
        self._tails = None

    def _plan(self):
        if self._specs is None:
            tp = self.time_proj
            t_w, t_b = (tp.weight, [tp.bias]) if isinstance(tp, nn.Linear) else (None, [])
            first = PlainLinear(self.d_model, [(self.input_proj.weight, self.input_proj.in_features),
                                               (t_w, self.d_time)], [self.input_proj.bias] + t_b)
            layers = []
            for l in self.transformer.layers:
                sa = l.self_attn
                layers.append((PlainLinear(3 * self.d_model, [(sa.in_proj_weight, self.d_model)], [sa.in_proj_bias]),
                               PlainLinear(self.d_model, [(sa.out_proj.weight, self.d_model)], [sa.out_proj.bias]),
                               PlainLinear(l.linear1.out_features, [(l.linear1.weight, self.d_model)], [l.linear1.bias]),
                               PlainLinear(self.d_model, [(l.linear2.weight, l.linear2.in_features)], [l.linear2.bias]),
                               l.norm1, l.norm2))
            self._specs = (first, layers)
        return self._specs

    def _tail_packs(self):
        """Parameter blocks of mmb_transformer_tail per layer (None when the widths are not compiled: d in {64, 128},
        FFN width a multiple of 64), rebuilt when a parameter changed."""
        d = self.d_model
        ls = list(self.transformer.layers)
        if os.environ.get("MMB_TR_TAIL") == "0" or d not in (64, 128) or not ls:
            return None
        ff = ls[0].linear1.out_features
        if ff % 64 or ff > 1024 or ls[0].activation_relu_or_gelu != 1 or ls[0].norm_first:
            return None
        key = tuple((q._version, q.data_ptr()) for l in ls for q in l.parameters())
        if self._tails is None or self._tails[0] != key:
            packs = [fused_epic.pack_transformer_tail(l, ls[i + 1] if i + 1 < len(ls) else None) for i, l in enumerate(ls)]
            self._tails = (key, packs)
        return self._tails[1]

    def run(self, ctx, time, x_segs, out=None, attn=None):
        """x_segs: list of (rows, SEG_ROW) whose widths add up to d_input.  Returns (B*N, d_model) rows (written into
        `out`, which may be a column slice, when given).  attn: replaces the attention (qkv rows -> attention output
        rows) -- the compacted inference path, where it is a gather of one V row per jet."""
        first, layers = self._plan()
        h = first.run(ctx, list(x_segs) + [_time_seg(time)])
        p = ctx.drop_p                                      # > 0 only in training mode (multimodal_epic._unpack)
        tails = self._tail_packs() if (not ctx.recording and p == 0.0) else None
        if tails is not None:
            # inference: attention, then ONE launch for out_proj + LN1 + FFN + LN2 + the next layer's in_proj
            # (csrc/transformer_fused.hip): h1 and the FFN's hidden tensor never reach HBM
            qkv = layers[0][0].run(ctx, [(h, SEG_ROW)]) if layers else None
            for i in range(len(layers)):
                last = i == len(layers) - 1
                if attn is not None:                       # compacted rows: the tail reads its jet's V row in place
                    h, qkv = fused_epic.transformer_tail(tails[i], qkv[:, 2 * self.d_model:], h, out=out if last else None,
                                                         want_qkv=not last, a_idx=attn.rows)
                    continue
                a = ops.attention_fwd(qkv, ctx.mi, self.n_heads, valid_is_zero=True)                 # quirk Q4
                h, qkv = fused_epic.transformer_tail(tails[i], a, h, out=out if last else None, want_qkv=not last)
            if not layers and out is not None:
                out.copy_(h)
                h = out
            return h
        kept = getattr(ctx, "kept", None) if ctx.recording else None
        for i, (in_proj, out_proj, lin1, lin2, norm1, norm2) in enumerate(layers):
            mark = len(ctx.tape) if kept is not None else 0
            qkv = in_proj.run(ctx, [(h, SEG_ROW)])
            rec = ctx.recording
            lse = rec and kept is None                     # (kept in 8 bits: the reverse pass runs the attention again)
            off = ctx.next_offset() if p > 0.0 else 0
            if attn is not None:
                r = attn(qkv)
            else:
                r = ops.attention_fwd(qkv, ctx.mi, self.n_heads, valid_is_zero=True, want_lse=lse,  # quirk Q4
                                      drop_p=p, seed=ctx.seed, offset=off)
            a = r[0] if lse else r
            if rec:
                ctx.tape.append(("attn", qkv, a, r[1] if lse else None, self.n_heads, p, off,
                                 r[2] if lse and len(r) > 2 else None))
            # x = norm1(x + dropout1(out_proj(attn)));  x = norm2(x + dropout2(linear2(dropout(relu(linear1(x))))))
            h1 = out_proj.run(ctx, [(a, SEG_ROW)], res1=h, norm=norm1, dropout=True)
            f = lin1.run(ctx, [(h1, SEG_ROW)], act="relu", dropout=True)
            h = lin2.run(ctx, [(f, SEG_ROW)], res1=h1, norm=norm2, out=out if i == len(layers) - 1 else None, dropout=True)
            if kept is not None:                           # all that this layer's entries hold, but its output
                for t, gate in activations(ctx.tape[mark:]):
                    if t is not h:
                        kept.keep(t, gate)
        if not layers and out is not None:
            out.copy_(h)
            h = out
        return h

    def forward(self, t_emb, x, mask):
        """Reference-style call: t_emb (B,N,d_time) per-particle (already masked), x (B,N,d_input), mask (B,N,1)."""
        ctx = ExecCtx(ops.mask_prepare(mask))
        rows = x.float().reshape(-1, x.shape[-1]).contiguous()
        h = self.run(ctx, t_emb.float().contiguous(), [(rows, SEG_ROW)])
        return h.view(ctx.B, ctx.N, -1)


class MultiModalParticleTransformer(nn.Module):
    """Two branch transformers (continuous / discrete features), an optional fusion transformer over cat[h1,h2]
    and two GELU MLP heads on cat[t, h_i, f_i] (particle_transformer.py:52-167)."""
    checkpoint_bits_choices = (None, 8)

    def __init__(self, config):
        super().__init__()
        self.config = config
        e, d = config.encoder, config.data
        self.checkpoint_bits = getattr(e, "checkpoint_bits", None)
        Et = e.dim_emb_time
        dim_cont, dim_disc = e.dim_emb_continuous, e.dim_emb_discrete * d.dim_discrete
        H0, H1 = e.dim_hidden_local[0], e.dim_hidden_local[1]
        nb = e.num_blocks
        ff = 4 * H0                                                   # particle_transformer.py:77
        kw = dict(d_time=Et, n_heads=e.num_heads, dim_feedforward=ff, dropout=e.dropout)
        self.continuous_encoder = TransformerEncoderBlock(d_input=dim_cont, d_model=H0, n_layers=nb[0], **kw)
        self.discrete_encoder = TransformerEncoderBlock(d_input=dim_disc, d_model=H1, n_layers=nb[1], **kw)
        self.mode_fusion = nb[2] > 0
        half = 0
        if self.mode_fusion:
            H2 = e.dim_hidden_local[2]
            self.fused_encoder = TransformerEncoderBlock(d_input=H0 + H1, d_model=H2, n_layers=nb[2], **kw)
            half = H2 // 2
        self.dims = (H0, H1, half)
        self.continuous_head = _Head(Et + H0 + half, H0, d.dim_continuous)
        self.discrete_head = _Head(Et + H1 + half, H1, d.vocab_size * d.dim_discrete)

    def run(self, ctx, time, cont, disc):
        H0, H1, half = self.dims
        M = ctx.B * ctx.N
        tseg = _time_seg(time)
        both = torch.empty(M, H0 + H1, dtype=torch.float32, device=cont.device)
        h1 = self.continuous_encoder.run(ctx, time, [(cont, SEG_ROW)], out=both[:, :H0])
        h2 = self.discrete_encoder.run(ctx, time, [(disc, SEG_ROW)], out=both[:, H0:])
        if self.mode_fusion:
            f = self.fused_encoder.run(ctx, time, [(both, SEG_ROW)])
            split = (f.shape[1] + 1) // 2                             # torch.chunk(fused, 2, dim=-1)
            hc = self.continuous_head.run(ctx, [tseg, (h1, SEG_ROW), (f[:, :split], SEG_ROW)])
            hd = self.discrete_head.run(ctx, [tseg, (h2, SEG_ROW), (f[:, split:], SEG_ROW)])
        else:
            hc = self.continuous_head.run(ctx, [tseg, (h1, SEG_ROW)])
            hd = self.discrete_head.run(ctx, [tseg, (h2, SEG_ROW)])
        return hc, hd

    def _compaction(self, state_local, ctx, time):
        """Row compaction of the inference path, or None.  The reference gives the attention the PADDED slots as keys
        (quirk Q4) and multiplies every input of the encoder by the mask (embedder.py:63-97), so in eval mode all padded
        slots of a jet carry the same row in every layer, every query's attention output is that row's V, and nothing
        else couples the rows of a jet: it is enough to run the real particles plus ONE padded slot per jet through the
        encoder and copy the representative's heads to the other padded slots (they ARE needed: padded slots are
        updated by the solvers, K3).  Only for the embedder's own factored state (LocalState: the masking is this
        package's, not the caller's), no tape, no dropout; at AOJ multiplicities (48 of 150 slots real on average) a
        third of the rows remain.  Row-wise kernels give every row the same bits wherever it sits."""
        if os.environ.get("MMB_TR_COMPACT") == "0" or not isinstance(state_local, LocalState) or \
                not isinstance(time, TimeSeg) or ctx.recording or ctx.drop_p > 0.0 or self.training:
            return None
        mi = ctx.mi
        cp = getattr(mi, "_compact", None)
        if cp is None:
            B, N = mi.B, mi.N
            mf = mi.maskf.reshape(-1)
            m = mf.view(B, N) > 0
            dev = m.device
            real = m.reshape(-1).nonzero().squeeze(1)                       # (one host sync per mask, i.e. per batch)
            has_pad = (~m).any(1)
            first_pad = (~m).to(torch.int8).argmax(1)
            rep_rows = (torch.arange(B, device=dev) * N + first_pad)[has_pad]
            rows = torch.cat([real, rep_rows])
            n_real, n_rep = int(real.numel()), int(rep_rows.numel())
            rep_c = torch.zeros(B, dtype=torch.int64, device=dev)
            rep_c[has_pad] = n_real + torch.arange(n_rep, device=dev)
            pos = rep_c.repeat_interleave(N)                                # padded slots -> their jet's representative
            pos[real] = torch.arange(n_real, device=dev)
            jet = torch.div(rows, N, rounding_mode="floor")
            src = torch.where(has_pad[jet], rep_c[jet], torch.full_like(jet, -1)).to(torch.int32)   # row -> its jet's V row
            cp = SimpleNamespace(rows=rows, jet=jet, src=src.contiguous(), all_pad=n_rep == B,
                                 has_pad=has_pad.float().unsqueeze(1), pos=pos, M=int(rows.numel()),
                                 maskf=mf.index_select(0, rows).contiguous())
            mi._compact = cp
        return cp if cp.M <= 0.85 * mi.B * mi.N else None

    def run_compact(self, ctx, time, cont, disc, cp):
        H0, H1, half = self.dims
        cctx = ExecCtx(SimpleNamespace(B=cp.M, N=1, maskf=cp.maskf, counts=None))
        t_rows = (time.temb.index_select(0, cp.jet) * cp.maskf.unsqueeze(1)).unsqueeze(0)     # (1, M', Et): explicit rows
        cont_c, disc_c = cont.index_select(0, cp.rows), disc.index_select(0, cp.rows)

        attn = _JetRowAttention(cp)

        both = torch.empty(cp.M, H0 + H1, dtype=torch.float32, device=cont.device)
        h1 = self.continuous_encoder.run(cctx, t_rows, [(cont_c, SEG_ROW)], out=both[:, :H0], attn=attn)
        h2 = self.discrete_encoder.run(cctx, t_rows, [(disc_c, SEG_ROW)], out=both[:, H0:], attn=attn)
        tseg = _time_seg(t_rows)
        if self.mode_fusion:
            f = self.fused_encoder.run(cctx, t_rows, [(both, SEG_ROW)], attn=attn)
            split = (f.shape[1] + 1) // 2
            hc = self.continuous_head.run(cctx, [tseg, (h1, SEG_ROW), (f[:, :split], SEG_ROW)])
            hd = self.discrete_head.run(cctx, [tseg, (h2, SEG_ROW), (f[:, split:], SEG_ROW)])
        else:
            hc = self.continuous_head.run(cctx, [tseg, (h1, SEG_ROW)])
            hd = self.discrete_head.run(cctx, [tseg, (h2, SEG_ROW)])
        return hc.index_select(0, cp.pos), hd.index_select(0, cp.pos)

    def forward(self, state_local, state_global=None, tape=None, seed=0, offset0=0) -> TensorMultiModal:
        glob = state_global if state_global is not None else TensorMultiModal(time=state_local.time)
        ctx, time, cont, disc, _ = _unpack(state_local, glob, self.training, self.config.encoder.dropout, tape, seed,
                                           offset0)
        if ctx.recording and self.checkpoint_bits:
            ctx.kept = Keep8()
            tape.append(("kept8", ctx.kept))
        cp = self._compaction(state_local, ctx, time)
        if cp is not None:
            hc, hd = self.run_compact(ctx, time, cont, disc, cp)
        else:
            hc, hd = self.run(ctx, time, cont, disc)
        B, N = ctx.B, ctx.N
        return TensorMultiModal(None, hc.view(B, N, -1), hd.view(B, N, -1), state_local.mask)
