"""GPU tests of the conditional transformer's operators against plain statements of them in 64 bits: cross attention
(forward, reverse), the norm of query and key heads with the rotation, 8-bit checkpoints and the weight gradient read from
them, and a run of all of them as a layer uses them.

Tolerances are bounds, not observations.  u(T) = eps(T) / 2 is the most one rounding to T is off, e = 2^-24 one 32-bit
rounding; a sum of n products in 32 bits is off by at most (n + 2) e times the sum of the products' magnitudes, the
exponential (hardware exp2 of a rounded argument) and the reciprocal by 2^-20 together.  Each reference returns, beside a
value, the magnitude that its bound scales with."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E = 2.0 ** -24
FN = 2.0 ** -20


def u(dt):
    return torch.finfo(dt).eps / 2


def out_step(dt, x):
    """One rounding of x to dt.  Half precision's step is never below 2^-24: half of that where x is subnormal."""
    return (u(dt) * x.abs()).clamp(min=2.0 ** -25 if dt == torch.float16 else 0.0)


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)                          # (a NaN is bad)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} x the bound"


# ------------------------------------------------------------------------------------------------ cross attention
def ref_attention(q, k, v, do, B, nh, nkv, mq, mk, scale, dt):
    """Values and bounds of out, lse, dq, dk, dv; all (B, n, heads, D) in 64 bits."""
    g, up = nh // nkv, (0.0 if dt == torch.float32 else u(dt))
    heads = lambda t, h: t.double().cpu().reshape(B, -1, h, t.shape[1] // h).permute(0, 2, 1, 3)  # noqa: E731
    q, do, k, v = heads(q, nh), heads(do, nh), heads(k, nkv), heads(v, nkv)
    Nq, Nk, D = q.shape[2], k.shape[2], q.shape[3]
    mq = torch.ones(B, Nq, dtype=torch.bool) if mq is None else mq.cpu() != 0
    mk = torch.ones(B, Nk, dtype=torch.bool) if mk is None else mk.cpu() != 0
    clean = lambda t, m: torch.where(m[:, None, :, None], t, 0.0)  # noqa: E731   what masked slots hold does not matter
    q, do, k, v = clean(q, mq), clean(do, mq), clean(k, mk), clean(v, mk)
    kr, vr = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = scale * q @ kr.transpose(2, 3)
    ok = (mq[:, :, None] & mk[:, None, :])[:, None]
    s = torch.where(ok, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    ex = torch.exp(s - top)
    z = ex.sum(-1, keepdim=True)
    p = torch.where(z > 0, ex / z, 0.0)
    lse = torch.where(z > 0, torch.log(z) + top, -math.inf).squeeze(-1)
    out = p @ vr
    # half precision: a p below 2^-14 of the row's largest is off by 2^-25 of that instead of relatively
    floor = 2.0 ** -25 if dt == torch.float16 else 0.0
    # p: error of a score twice (its own and the sum's), the sums' roundings, the functions
    S = float((scale * q.abs() @ kr.abs().transpose(2, 3)).max()) if s.numel() else 0.0
    ep = 2 * (D + 4) * E * S + Nk * E + FN
    t_out = (p @ vr.abs()) * (ep + up + (Nk + 2) * E) + out_step(dt, out) + 1e-30 + floor * p.amax(-1, keepdim=True) * vr.abs().sum(2, keepdim=True)
    t_lse = (ep + 4 * E * top.abs().squeeze(-1) + FN)
    dp, dpa = do @ vr.transpose(2, 3), do.abs() @ vr.abs().transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (do.abs() * t_out).sum(-1, keepdim=True) + (D + 2) * E * (do.abs() * out.abs()).sum(-1, keepdim=True)
    e_ds = p * ((ep + 4 * E * S) * (dpa + delta.abs()) + (D + 2) * E * dpa + e_delta) + up * ds.abs()
    sum_g = lambda t: t.reshape(B, nkv, g, Nk, D).sum(2)  # noqa: E731
    pt, rows = p.transpose(2, 3), g * Nq
    dv, dq, dk = sum_g(pt @ do), scale * ds @ kr, scale * sum_g(ds.transpose(2, 3) @ q)
    t_dv = sum_g(pt @ do.abs()) * (ep + 4 * E * S + up + (rows + 2) * E) + out_step(dt, dv) + 1e-30
    t_dq = scale * (e_ds @ kr.abs() + (Nk + 2) * E * ds.abs() @ kr.abs()) + out_step(dt, dq) + 1e-30
    t_dk = scale * (sum_g(e_ds.transpose(2, 3) @ q.abs()) + (rows + 2) * E * sum_g(ds.abs().transpose(2, 3) @ q.abs())) + out_step(dt, dk) + 1e-30
    flat = lambda t: t.permute(0, 2, 1, 3).reshape(t.shape[0] * t.shape[2], -1)  # noqa: E731
    return {"out": (flat(out), flat(t_out)), "lse": (lse, t_lse.expand_as(lse) if not torch.is_tensor(t_lse) else t_lse),
            "dq": (flat(dq), flat(t_dq)), "dk": (flat(dk), flat(t_dk)), "dv": (flat(dv), flat(t_dv))}


def slots(B, N, g, empty=True):
    n = torch.randint(0 if empty else 1, N + 1, (B,), generator=g)
    n[0] = N
    if B > 1 and empty:
        n[1] = 0
    return (torch.rand(B, N, generator=g).argsort(1).argsort(1) < n[:, None]).float()


def make(B, Nq, Nk, nh, nkv, D, dt, seed, masked, size=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = ((size * torch.randn(B * n, h * D, generator=g)).to(dt) for n, h in ((Nq, nh), (Nk, nkv), (Nk, nkv), (Nq, nh)))
    mq, mk = (slots(B, Nq, g), slots(B, Nk, g)) if masked else (None, None)
    return q, k, v, do, mq, mk


def run_attention(q, k, v, do, mq, mk, B, nh, nkv, scale):
    from mmb_hip import ops
    info = lambda m: None if m is None else ops.mask_prepare(m.cuda())  # noqa: E731
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    kw = dict(nheads_kv=nkv, mq=info(mq), mk=info(mk), scale=scale)
    out, lse = ops.cross_attention_fwd(q, k, v, B, nh, want_lse=True, **kw)
    dq, dk, dv = ops.cross_attention_bwd(q, k, v, out, do, lse, B, nh, **kw)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def check_attention(got, ref):
    lse, want = got["lse"].double().cpu(), ref["lse"][0]
    assert torch.equal(lse == -math.inf, want == -math.inf)
    fin = want > -math.inf
    within(lse[fin], want[fin], ref["lse"][1][fin], "lse")
    for n in ("out", "dq", "dk", "dv"):
        within(got[n], *ref[n], n)


SHAPES = [  # B, Nq, Nk, nh, nkv, D, masked
    (1, 1, 1, 1, 1, 16, False),
    (2, 1, 150, 4, 4, 16, True),
    (3, 128, 150, 4, 4, 32, True),
    (2, 150, 31, 4, 2, 16, True),
    (2, 33, 65, 6, 2, 64, False),
    (1, 257, 300, 3, 1, 128, True),
    (2, 7, 1000, 8, 2, 128, True),
    (1, 3, 2500, 10, 2, 64, True),                              # one row tile, keys split over workgroups
    (1, 40, 1500, 2, 1, 80, False),                             # a few row tiles, split
    (9, 64, 64, 5, 5, 20, True),
    (8, 100, 96, 2, 1, 33, True),                               # odd head width: scalar loads
    (2, 130, 70, 3, 3, 1, False),
    (4, 5, 600, 4, 4, 8, True),
    (5, 2, 300, 15, 3, 16, True),                               # few queries: the heads of a group share tiles
    (3, 9, 130, 20, 2, 32, True),
    (2, 1, 100, 70, 1, 8, False),
    (64, 150, 128, 4, 4, 16, True),                             # many small clouds: their keys stay in LDS
    (70, 40, 50, 8, 4, 32, True),
    (128, 16, 20, 4, 2, 64, True),
    (300, 33, 150, 2, 1, 12, True),
    (256, 20, 40, 1, 1, 128, False),
    (66, 17, 200, 4, 4, 21, True),
    (500, 18, 1, 2, 2, 8, False),
    (256, 130, 150, 2, 2, 128, True),                           # eight waves share a tile
    (65, 66, 2562, 4, 4, 16, True),                             # keys in two ranges
    (65, 33, 2561, 8, 4, 40, False),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(str(int(v)) for v in s) for s in SHAPES])
def test_cross_attention(shape, dtype):
    B, Nq, Nk, nh, nkv, D, masked = shape
    dt = TYPES[dtype]
    args = make(B, Nq, Nk, nh, nkv, D, dt, sum(shape) + Nk, masked)
    scale = 1.0 / math.sqrt(D)
    check_attention(run_attention(*args, B, nh, nkv, scale), ref_attention(*args[:4], B, nh, nkv, *args[4:], scale, dt))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_cross_attention_peaked_scores(dtype):
    """Large scores: one key takes almost everything, the running maximum jumps from tile to tile."""
    dt = TYPES[dtype]
    args = make(2, 70, 700, 2, 1, 64, dt, 5, True, size=3.0)
    check_attention(run_attention(*args, 2, 2, 1, 1.0), ref_attention(*args[:4], 2, 2, 1, *args[4:], 1.0, dt))


def test_cross_attention_reverse_leaves_masked_queries_unread():
    """The workspace of the reverse holds dout . out of every (cloud, head, query): nothing is found out for masked ones."""
    import mmb_hip
    from mmb_hip import ops
    B, Nq, Nk, nh, D = 3, 37, 90, 2, 16
    q, k, v, do, mq, mk = (t.cuda() for t in make(B, Nq, Nk, nh, nh, D, torch.float32, 13, True))
    out, lse = ops.cross_attention_fwd(q, k, v, B, nh, mq=ops.mask_prepare(mq), mk=ops.mask_prepare(mk), want_lse=True)
    grads, ws = [torch.empty_like(t) for t in (q, k, v)], torch.full((B, nh, Nq), 123.0, device="cuda")
    ld = nh * D
    mmb_hip.call("mmb_cross_attention_bwd", B, Nq, Nk, nh, nh, D, 0, q.data_ptr(), ld, k.data_ptr(), ld, v.data_ptr(), ld,
                 ops.f32(mq.reshape(-1)), ops.f32(mk.reshape(-1)), D ** -0.5, out.data_ptr(), ld, do.data_ptr(), ld, ops.f32(lse),
                 grads[0].data_ptr(), ld, grads[1].data_ptr(), ld, grads[2].data_ptr(), ld, ws.data_ptr(), ws.numel() * 4, ops.stream())
    gone = (mq == 0)[:, None].expand(B, nh, Nq)
    assert gone.any() and bool((ws[gone] == 123.0).all())
    kept = (do * out).view(B, Nq, nh, D).sum(-1).transpose(1, 2)[~gone]
    torch.testing.assert_close(ws[~gone], kept, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Nq,Nk", [(40, 50), (2, 900)])
def test_cross_attention_masked_slots_hold_anything(dtype, Nq, Nk):
    """NaN, infinities and the type's largest values in padded rows change no bit."""
    dt = TYPES[dtype]
    B, nh, nkv, D = 3, 4, 2, 32
    q, k, v, do, mq, mk = make(B, Nq, Nk, nh, nkv, D, dt, 11, True)
    clean = run_attention(q, k, v, do, mq, mk, B, nh, nkv, 0.3)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dt).max, torch.finfo(dt).min):
        dirty = [torch.where(m.reshape(-1, 1) != 0, t, torch.tensor(bad, dtype=dt)) for t, m in ((q, mq), (k, mk), (v, mk), (do, mq))]
        got = run_attention(*dirty, mq, mk, B, nh, nkv, 0.3)
        for n in clean:
            assert torch.equal(got[n], clean[n]), (bad, n)
    gone = (mq == 0).reshape(-1)
    assert gone.any() and not got["out"][gone.cuda()].any() and not got["dq"][gone.cuda()].any()
    gone = (mk == 0).reshape(-1)
    assert not got["dk"][gone.cuda()].any() and not got["dv"][gone.cuda()].any()
    assert not got["out"][Nq:2 * Nq].any()                      # the cloud without a key


@pytest.mark.parametrize("Nk,at", [(40, (17, 39)), (20, (0, 19))])
def test_cross_attention_single_key(Nk, at):
    """One kept key: out is its value row.  dq and dk are zero: exactly with up to 32 slots, where delta comes from the row's
    own p and dp; else to what dp and delta = do . o -- the same D products, summed in 32 bits in two orders, so at most
    2 (D + 2) e times the sum of their magnitudes apart -- leave of each other (p = 1 to FN; half precision adds its step)."""
    B, Nq, nh, nkv, D = 2, 9, 4, 2, 64
    for dt in TYPES.values():
        q, k, v, do, _, _ = make(B, Nq, Nk, nh, nkv, D, dt, 3, False)
        mk = torch.zeros(B, Nk)
        mk[0, at[0]], mk[1, at[1]] = 1, 1
        got = run_attention(q, k, v, do, None, mk, B, nh, nkv, 0.125)
        one = lambda t: torch.stack([t.view(B, Nk, nkv, D)[b, s] for b, s in enumerate(at)]).repeat_interleave(nh // nkv, 1)  # noqa: E731
        assert torch.equal(got["out"].cpu().view(B, Nq, nh, D), one(v)[:, None].expand(B, Nq, nh, D))
        if Nk <= 32:
            assert not got["dq"].any() and not got["dk"].any()
            continue
        ds = 2 * (D + 2) * E * (do.double().view(B, Nq, nh, D).abs() * one(v).double().abs()[:, None]).sum(-1, keepdim=True) * (1 + FN)
        ds = ds * (1 + u(dt))                                   # (its rounding for the product)
        t_dq = 0.125 * ds * one(k).double().abs()[:, None]
        t_dk = 0.125 * (ds * q.double().view(B, Nq, nh, D).abs()).view(B, Nq, nkv, nh // nkv, D).sum((1, 3))
        within(got["dq"].view(B, Nq, nh, D), torch.zeros(B, Nq, nh, D).double(), t_dq + out_step(dt, t_dq) + 1e-30, "dq")
        dk = got["dk"].view(B, Nk, nkv, D)
        within(torch.stack([dk[b, s] for b, s in enumerate(at)]), torch.zeros_like(t_dk), t_dk + out_step(dt, t_dk) + 1e-30, "dk")
        assert not dk[0, :at[0]].any() and not dk[1, :at[1]].any()


@pytest.mark.parametrize("B,Nq,Nk,nh,D", [(1, 300, 16384, 1, 16), (1, 1, 16384, 2, 64), (2, 130, 3000, 4, 128), (260, 20, 128, 1, 32), (64, 300, 700, 4, 33)])
def test_cross_attention_long_tail_of_small_probabilities(B, Nq, Nk, nh, D):
    """One key takes nearly all of a row, the others e^-18 = 2^-26 of it each: less than half of half precision's smallest step,
    but together Nk times that.  Values are 0 at the strong key and 1024 or 2048 at the others, so the output is the tail alone.
    Bound: p of the tail is off by one rounding to half (u), its exponent by the rounding of 18 log2(e) and of the row's offset
    (4 x 64 E), sums of Nk terms by Nk E each in numerator and denominator; the output's own rounding."""
    dt = torch.float16
    at = Nk // 3
    q, k, v = torch.zeros(B * Nq, nh * D), torch.zeros(B * Nk, nh * D), torch.full((B * Nk, nh * D), 1024.0)
    v[1::2] = 2048.0
    q.view(-1, nh, D)[:, :, 0] = 1.0
    k.view(B, Nk, nh, D)[:, at, :, 0] = 18.0
    v.view(B, Nk, nh * D)[:, at] = 0.0
    got = run_attention(*(t.to(dt) for t in (q, k, v, torch.zeros_like(q))), None, None, B, nh, nh, 1.0)
    tail = math.exp(-18.0)
    tot = v.view(B, Nk, nh * D)[0, :, 0].double().sum() * tail
    den = 1.0 + (Nk - 1) * tail
    want = torch.full((B * Nq, nh * D), float(tot) / den, dtype=torch.float64)
    within(got["out"], want, (u(dt) + 256 * E + 2 * (Nk + 2) * E + FN) * want + out_step(dt, want), "out")
    lse = torch.full((B, nh, Nq), 18.0 + math.log(den), dtype=torch.float64)
    within(got["lse"], lse, torch.full_like(lse, 4 * 18 * E + FN + (Nk + 2) * E), "lse")


def test_cross_attention_values_that_are_not_finite():
    """A NaN in a kept key spoils the clouds and heads that see it and no others; scores of -inf take no weight."""
    B, Nq, Nk, nh, D = 2, 5, 40, 2, 16
    q, k, v, do, _, _ = make(B, Nq, Nk, nh, nh, D, torch.float32, 8, False)
    base = run_attention(q, k, v, do, None, None, B, nh, nh, 0.25)["out"].view(B, Nq, nh, D)
    k2 = k.clone()
    k2[3, 2] = math.nan                                         # cloud 0, head 0
    got = run_attention(q, k2, v, do, None, None, B, nh, nh, 0.25)["out"].view(B, Nq, nh, D)
    assert got[0, :, 0].isnan().all() and torch.equal(got[1], base[1]) and torch.equal(got[0, :, 1], base[0, :, 1])
    q3, k3 = q.abs() + 0.1, k.clone()
    k3[:Nk, :D] = -math.inf                                     # every score of cloud 0, head 0 is -inf: no weight at all
    got = run_attention(q3, k3, v, do, None, None, B, nh, nh, 0.25)
    assert not got["out"].view(B, Nq, nh, D)[0, :, 0].any() and got["lse"][0, 0].eq(-math.inf).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("off", [0, 1])
def test_cross_attention_strides_and_what_lies_around(dtype, off):
    """Column slices of wider rows, aligned (off 0) and not (off 1); nothing outside the outputs is written."""
    from mmb_hip import ops
    dt = TYPES[dtype]
    B, Nq, Nk, nh, nkv, D = 2, 45, 77, 4, 2, 32
    q, k, v, do, mq, mk = make(B, Nq, Nk, nh, nkv, D, dt, 21, True)
    dense = run_attention(q, k, v, do, mq, mk, B, nh, nkv, 0.2)

    def wide(t, fill=None):
        w = torch.full((t.shape[0] + 3, t.shape[1] + 24), 7.0, dtype=dt, device="cuda")
        view = w[1:1 + t.shape[0], 8 + off:8 + off + t.shape[1]]
        if fill is None:
            view.copy_(t)
        return w, view

    mqi, mki = ops.mask_prepare(mq.cuda()), ops.mask_prepare(mk.cuda())
    (_, qv), (_, kv), (_, vv), (_, gv) = wide(q), wide(k), wide(v), wide(do)
    outs = {n: wide(t, fill=0) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    _, lse = ops.cross_attention_fwd(qv, kv, vv, B, nh, nkv, mqi, mki, 0.2, True, outs["out"][1])
    ops.cross_attention_bwd(qv, kv, vv, outs["out"][1], gv, lse, B, nh, nkv, mqi, mki, 0.2, outs["dq"][1], outs["dk"][1], outs["dv"][1])
    for n, (w, view) in outs.items():
        assert torch.equal(view, dense[n]), n                   # the same arithmetic: the same bits
        rest = w.clone()
        rest[1:1 + view.shape[0], 8 + off:8 + off + view.shape[1]] = 7.0
        assert bool((rest == 7.0).all()), n


def test_cross_attention_all_in_the_columns_of_one_matrix():
    """Inputs, output and gradients side by side in the same rows share no memory: the call is taken and gives the same bits."""
    from mmb_hip import ops
    B, N, nh, D = 2, 70, 2, 16
    q, k, v, do, mq, mk = make(B, N, N, nh, nh, D, torch.float32, 51, True)
    want = run_attention(q, k, v, do, mq, mk, B, nh, nh, 0.25)
    w = torch.full((B * N, 8 * 32 + 5), 3.0, device="cuda")
    c = [w[:, 32 * i:32 * i + 32] for i in range(8)]
    for t, x in zip(c, (q, k, v, do)):
        t.copy_(x)
    kw = dict(mq=ops.mask_prepare(mq.cuda()), mk=ops.mask_prepare(mk.cuda()), scale=0.25)
    _, lse = ops.cross_attention_fwd(*c[:3], B, nh, want_lse=True, out=c[4], **kw)
    ops.cross_attention_bwd(*c[:3], c[4], c[3], lse, B, nh, dq=c[5], dk=c[6], dv=c[7], **kw)
    for t, n in zip(c[4:], ("out", "dq", "dk", "dv")):
        assert torch.equal(t, want[n]), n
    assert all(torch.equal(t.cpu(), x) for t, x in zip(c, (q, k, v, do))) and bool((w[:, 256:] == 3.0).all())


def test_cross_attention_equal_bits_and_clouds_alone():
    """The same call twice, and each cloud in a call of its own, give equal bits."""
    args = make(3, 90, 400, 4, 2, 64, torch.bfloat16, 31, True)
    a, b = (run_attention(*args, 3, 4, 2, 0.125) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)
    q, k, v, do, mq, mk = args
    for c in range(3):
        one = run_attention(*(t[c * n:(c + 1) * n] for t, n in ((q, 90), (k, 400), (v, 400), (do, 90))), mq[c:c + 1], mk[c:c + 1], 1, 4, 2, 0.125)
        # (one cloud alone may split its keys: another order of the sum over keys in out; the reverse has one form)
        want = ref_attention(*(t[c * n:(c + 1) * n] for t, n in ((q, 90), (k, 400), (v, 400), (do, 90))), 1, 4, 2, mq[c:c + 1], mk[c:c + 1], 0.125, torch.bfloat16)
        check_attention(one, want)


def test_cross_attention_offsets_past_32_bits():
    """Keys whose addresses lie further than 2^32 elements apart."""
    from mmb_hip import ops
    Nk, D, ld = 4200, 64, 1 << 20
    g = torch.Generator().manual_seed(4)
    big = torch.empty(Nk * ld, dtype=torch.bfloat16, device="cuda").view(Nk, ld)
    k, v, q, do = (torch.randn(n, D, generator=g).bfloat16() for n in (Nk, Nk, 20, 20))
    kw, vw = big[:, :D], big[:, 512:512 + D]
    kw.copy_(k)
    vw.copy_(v)
    out, lse = ops.cross_attention_fwd(q.cuda(), kw, vw, 1, 1, want_lse=True)
    dkw, dvw = big[:, 1024:1024 + D], big[:, 2048:2048 + D]
    dq, _, _ = ops.cross_attention_bwd(q.cuda(), kw, vw, out, do.cuda(), lse, 1, 1, dk=dkw, dv=dvw)
    check_attention({"out": out, "lse": lse, "dq": dq, "dk": dkw, "dv": dvw},
                    ref_attention(q, k, v, do, 1, 1, 1, None, None, D ** -0.5, torch.bfloat16))


def test_gradients_against_differences():
    """d loss / d input along random directions, by central differences of the 64-bit forward, at one small shape."""
    B, Nq, Nk, nh, nkv, D = 2, 6, 9, 4, 2, 8
    q, k, v, do, mq, mk = make(B, Nq, Nk, nh, nkv, D, torch.float32, 41, True)
    got = run_attention(q, k, v, do, mq, mk, B, nh, nkv, 0.4)
    g = torch.Generator().manual_seed(1)
    f = lambda q, k, v: (ref_attention(q, k, v, do, B, nh, nkv, mq, mk, 0.4, torch.float32)["out"][0] * do.double()).sum()  # noqa: E731
    for i, n in enumerate(("dq", "dk", "dv")):
        x = [q.double(), k.double(), v.double()]
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + h * d, x[i] - h * d
        want = (f(*hi) - f(*lo)) / (2 * h)
        have = (got[n].double().cpu() * d).sum()
        # difference quotient: O(h^2) and 2^-52 / h; the gradient itself: 2^-18 of its magnitude (32-bit sums of <= 64 terms)
        assert abs(float(want - have)) <= 2 ** -18 * float((got[n].double().cpu().abs() * d.abs()).sum()) + 1e-7


# ------------------------------------------------------------------------------------------------ head norm and rotation
def ref_head_norm(x, dy, nh, w1, nh2, w2, eps, pos, freq, layout, dt):
    M, H = x.shape[0], nh + nh2
    D = x.shape[1] // H
    x = x.double().cpu().view(M, H, D)
    one = torch.ones(D, dtype=torch.float64)
    ws = torch.stack([one if w is None else w.double().cpu() for w in [w1] * nh + [w2] * nh2])
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = x * r
    P = 0 if freq is None else freq.numel()
    i = torch.arange(P) if layout == "half" else 2 * torch.arange(P)
    j = i + P if layout == "half" else i + 1
    if P:
        ang = pos.double().cpu().repeat_interleave(P // pos.shape[1], 1) * freq.double().cpu()
        c, s = ang.cos()[:, None], ang.sin()[:, None]

    def turn(t, sg):
        t, m = t.clone(), t.abs()
        if P:
            a, b = t[..., i].clone(), t[..., j].clone()
            t[..., i], t[..., j] = a * c - sg * b * s, sg * a * s + b * c
            m[..., i] = m[..., j] = a.abs() + b.abs()
        return t, m

    y, ym = turn(hat * ws, 1.0)
    # r: a sum of D squares under a root; the angle: a 32-bit fraction of a turn; three products
    er = (D / 2 + 8) * E + 2.0 ** -21
    t_y = er * ym + out_step(dt, y) + 1e-30
    g, gm = turn(dy.double().cpu().view(M, H, D), -1.0)
    dot, dota = (g * ws * hat).mean(-1, keepdim=True), (gm * ws.abs() * hat.abs()).mean(-1, keepdim=True)
    dx = r * (g * ws - hat * dot)
    t_dx = r * (gm * ws.abs() + hat.abs() * dota) * (3 * er + (D + 8) * E) + out_step(dt, dx) + 1e-30
    dw, dwm = (g * hat).sum(0), (gm * hat.abs()).sum(0)
    n = M * H
    two = lambda t: (t[:nh].sum(0), t[nh:].sum(0))  # noqa: E731
    flat = lambda t: t.reshape(M, -1)  # noqa: E731
    tw = [m * (2 * er + (n + 2) * E) + 1e-30 for m in two(dwm)]
    return {"y": (flat(y), flat(t_y)), "dx": (flat(dx), flat(t_dx)), "dw1": (two(dw)[0], tw[0]), "dw2": (two(dw)[1], tw[1])}


NORMS = [  # M, nheads, nheads2, D, pairs, axes, layout, far
    (1, 1, 0, 8, 0, 1, "half", 1.0),
    (5, 2, 1, 32, 16, 1, "half", 1e5),
    (150, 4, 4, 32, 16, 2, "interleaved", 3.2),
    (33, 8, 2, 128, 64, 1, "half", 1e6),
    (200, 3, 0, 64, 16, 2, "half", 4096.0),
    (70, 1, 2, 128, 32, 1, "interleaved", 1e5),
    (40, 2, 2, 80, 40, 1, "half", 100.0),
    (17, 3, 1, 96, 12, 3, "interleaved", 10.0),
    (29, 2, 0, 20, 10, 2, "half", 50.0),                        # widths and pairs off the chunk: one wave a head
    (12, 1, 1, 33, 16, 1, "interleaved", 3e4),
    (9, 2, 1, 256, 128, 1, "half", 1e5),
    (6, 1, 0, 1, 0, 1, "half", 1.0),
    (5000, 2, 1, 16, 8, 2, "half", 3.2),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", NORMS, ids=["x".join(str(v) for v in c[:6]) + c[6] for c in NORMS])
def test_head_norm_rotate(case, dtype):
    from mmb_hip import ops
    M, nh, nh2, D, P, A, layout, far = case
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M + D + P)
    x, dy = (torch.randn(M, (nh + nh2) * D, generator=g).to(dt) for _ in range(2))
    x[0] = 0                                                    # a row of zeros: eps alone
    w1, w2 = 1 + 0.3 * torch.randn(D, generator=g), (torch.randn(D, generator=g) if nh2 else None)
    pos = far * (2 * torch.rand(M, A, generator=g) - 1) if P else None
    freq = torch.rand(P, generator=g) if P else None
    if P:
        freq[0] = 1.0
    eps = 1e-5
    ref = ref_head_norm(x, dy, nh, w1, nh2, w2, eps, pos, freq, layout, dt)
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    kw = dict(nheads2=nh2, weight2=cu(w2), eps=eps, pos=cu(pos), freq=cu(freq), layout=layout)
    xd, gd = x.cuda(), dy.cuda()
    y = ops.head_norm_rotate_fwd(xd, nh, cu(w1), **kw)
    within(y, *ref["y"], "y")
    dx, d1, d2 = ops.head_norm_rotate_bwd(xd, gd, nh, cu(w1), **kw)
    within(dx, *ref["dx"], "dx")
    within(d1, *ref["dw1"], "dweight")
    assert (d2 is None) == (w2 is None)
    if nh2:
        within(d2, *ref["dw2"], "dweight2")
    again = ops.head_norm_rotate_bwd(xd, gd, nh, cu(w1), **kw)
    assert torch.equal(again[0], dx) and torch.equal(again[1], d1)
    # in place, both ways; no weight
    z = xd.clone()
    assert torch.equal(ops.head_norm_rotate_fwd(z, nh, cu(w1), out=z, **kw), y)
    z = gd.clone()
    assert torch.equal(ops.head_norm_rotate_bwd(xd, z, nh, cu(w1), dx=z, **kw)[0], dx)
    kw["weight2"] = None
    within(ops.head_norm_rotate_fwd(xd, nh, None, **kw), *ref_head_norm(x, dy, nh, None, nh2, None, eps, pos, freq, layout, dt)["y"], "no weight")


@pytest.mark.parametrize("D", [32, 33])
def test_head_norm_rotate_reverse_over_its_input(D):
    """dx may be x: every head is read whole before its gradient is written."""
    from mmb_hip import ops
    g = torch.Generator().manual_seed(D)
    x, dy, w = torch.randn(300, 3 * D, generator=g).cuda(), torch.randn(300, 3 * D, generator=g).cuda(), torch.rand(D, generator=g).cuda()
    kw = dict(pos=torch.randn(300, 1, generator=g).cuda(), freq=torch.rand(16, generator=g).cuda())
    dx, dw, _ = ops.head_norm_rotate_bwd(x, dy, 3, w, **kw)
    z = x.clone()
    got, dw2, _ = ops.head_norm_rotate_bwd(z, dy, 3, w, dx=z, **kw)
    assert got is z and torch.equal(z, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("off", [0, 1])
def test_head_norm_rotate_slices(dtype, off):
    """q and k of packed [q | k | v] rows, positions as two columns of a wider state; aligned and not."""
    from mmb_hip import ops
    dt, M, D = TYPES[dtype], 37, 32
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(M, 6 * D + 8, generator=g).to(dt).cuda()
    state = torch.randn(M, 3, generator=g).cuda()
    freq, w = torch.rand(16, generator=g).cuda(), torch.rand(D, generator=g).cuda()
    kw = dict(nheads2=2, weight2=w, pos=state[:, 1:], freq=freq, layout="interleaved")
    x = wide[:, off:off + 4 * D]
    want = ops.head_norm_rotate_fwd(x.contiguous(), 2, w, **kw)
    keep = wide.clone()
    ops.head_norm_rotate_fwd(x, 2, w, out=x, **kw)
    within(x, want.double().cpu(), (4 * u(dt) + 2.0 ** -18) * want.double().cpu().abs() + 1e-6, "slice")
    keep[:, off:off + 4 * D] = x
    assert torch.equal(keep, wide)


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints
def ref_codes(x):
    M, K = x.shape
    nb = -(-K // 32)
    xb = torch.zeros(M, nb * 32, dtype=torch.float64)
    xb[:, :K] = x.double().cpu()
    xb = xb.view(M, nb, 32)
    top = xb.abs().amax(-1)
    e = torch.full((M, nb), -127, dtype=torch.int64)
    for _ in range(260):
        e += (127.0 * torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double()) < top).long()
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())
    codes = torch.round(xb / step[..., None])
    return codes.view(M, -1), e, (codes * step[..., None]).view(M, -1)[:, :K]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (3, 32), (150, 64), (77, 100), (19, 33), (260, 128), (5, 1000)])
def test_checkpoint_rows(dtype, M, K):
    from mmb_hip import ops
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-12, 12, (M, 1), generator=g).float())
    x = x.to(dt)
    x[0] = 0
    if K >= 32 and M > 2:                                       # exactly on, just under and just over the codes' range; ties
        x[1, :32] = 0
        x[1, 0], x[1, 1], x[1, 2] = 127.0, 0.5, 1.5
        x[2, :32] = 0
        x[2, 0], x[2, 1] = 128.0, 3.0
    codes, e, val = ref_codes(x)
    q8 = ops.checkpoint_rows(x.cuda())
    assert torch.equal(q8.codes.double().cpu(), codes) and torch.equal(q8.steps.long().cpu() - 127, e)
    for out_t in TYPES.values():
        assert torch.equal(ops.restore_rows(q8, out_t).cpu(), val.to(out_t))
    assert bool(((val - x.double()).abs() <= 0.5 * torch.exp2(e.double()).repeat_interleave(32, 1)[:, :K]).all())
    # a slice of wider rows (not aligned), restored into another
    wide = torch.zeros(M, K + 5, dtype=dt, device="cuda")
    wide[:, 3:3 + K] = x.cuda()
    q2 = ops.checkpoint_rows(wide[:, 3:3 + K])
    assert torch.equal(q2.codes, q8.codes) and torch.equal(q2.steps, q8.steps)
    back = torch.full((M, K + 5), 9.0, device="cuda")
    ops.restore_rows(q8, out=back[:, 1:1 + K])
    assert torch.equal(back[:, 1:1 + K].cpu(), val.float()) and bool((back[:, 0] == 9).all()) and bool((back[:, 1 + K:] == 9).all())


def test_checkpoint_keeps_nonzero_values():
    """keep_nonzero: the sign of every value survives, whatever its size beside the block's largest; all else is the same."""
    from mmb_hip import ops
    g = torch.Generator().manual_seed(9)
    x = torch.randn(60, 96, generator=g) * torch.exp2(torch.randint(-40, 4, (60, 96), generator=g).float())
    x[:, ::7] = 0
    x[0, :32], x[1, 32:64] = 0, 2.0 ** -149
    plain, kept = ops.checkpoint_rows(x.cuda()), ops.checkpoint_rows(x.cuda(), keep_nonzero=True)
    assert torch.equal(plain.steps, kept.steps)
    y = ops.restore_rows(kept).cpu()
    assert torch.equal(kept.codes.cpu().sign().float(), x.sign())
    zero = plain.codes == 0
    assert bool(zero.any()) and torch.equal(plain.codes[~zero], kept.codes[~zero])
    step = torch.exp2(kept.steps.double().cpu() - 127).repeat_interleave(32, 1)
    assert bool(((y.double() - x.double()).abs() < step).all())


def test_checkpoint_extremes():
    from mmb_hip import ops
    big = torch.finfo(torch.float32).max
    x = torch.zeros(8, 64)
    x[0, 0], x[0, 1] = big, -big                                # stays finite
    x[1, 0], x[1, 40] = 2.0 ** -149, 2.0 ** -130                # subnormal
    x[2, 5], x[3, 5], x[4, 37] = math.nan, math.inf, -math.inf  # the block is NaN, its neighbour is not
    x[2:5, 0], x[2:5, 63] = 1.0, 2.0
    y = ops.restore_rows(ops.checkpoint_rows(x.cuda())).cpu()
    assert y[0].isfinite().all() and abs(float(y[0, 0]) / big - 1) <= 2.0 ** -6 and float(y[0, 1]) == -float(y[0, 0])
    assert abs(float(y[1, 40]) - 2.0 ** -130) <= 2.0 ** -128 and float(y[1, 0]) == 0.0
    for r, lo in ((2, 0), (3, 0), (4, 32)):
        assert y[r, lo:lo + 32].isnan().all() and y[r, 32 - lo:64 - lo].isfinite().all()
    top = torch.tensor([[65504.0, -65504.0, 1.0]], dtype=torch.float16)
    assert ops.restore_rows(ops.checkpoint_rows(top.cuda()), torch.float16).isfinite().all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (5, 32, 4), (150, 64, 192), (1000, 128, 384), (777, 100, 33), (4097, 256, 130), (33, 1000, 7),
                                   (20000, 64, 64)])
def test_grad_weight_rows_q8(dtype, M, K, N):
    from mmb_hip import ops
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M + K + N)
    q8 = ops.checkpoint_rows((torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).cuda())
    dz = torch.randn(M, N, generator=g).to(dt)
    x, z = ops.restore_rows(q8).double().cpu(), dz.double()
    dW, db = ops.grad_weight_rows_q8(q8, dz.cuda())
    tol = (M + 4) * E * (z.abs().t() @ x.abs()) + 1e-30         # exact products, a 32-bit sum of M terms
    within(dW, z.t() @ x, tol, "dW")
    within(db, z.sum(0), (M + 4) * E * z.abs().sum(0) + 1e-30, "db")
    again = ops.grad_weight_rows_q8(q8, dz.cuda())
    assert torch.equal(again[0], dW) and torch.equal(again[1], db)
    # added to what is there, into a column slice, from a slice of wider rows
    wide, b0 = torch.ones(N, K + 3, device="cuda"), torch.ones(N, device="cuda")
    zw = torch.zeros(M, N + 3, dtype=dt, device="cuda")
    zw[:, 1:1 + N] = dz.cuda()
    ops.grad_weight_rows_q8(q8, zw[:, 1:1 + N], dW=wide[:, 2:2 + K], db=b0, accumulate=True)
    assert torch.equal(wide[:, 2:2 + K], 1 + dW) and torch.equal(b0, 1 + db)
    assert bool((wide[:, :2] == 1).all()) and bool((wide[:, 2 + K:] == 1).all())
    only, none = ops.grad_weight_rows_q8(q8, dz.cuda(), want_db=False)
    assert none is None and torch.equal(only, dW)


def test_grad_weight_rows_q8_extremes():
    """Codes of the largest floats and of subnormals; a block that was not finite spoils its own columns of dW and no others."""
    from mmb_hip import ops
    x = torch.zeros(40, 96)
    x[:, 0], x[:, 1], x[:, 33] = torch.finfo(torch.float32).max, -1.0e38, 2.0 ** -140
    dz = torch.full((40, 8), 2.0 ** -20)
    q8 = ops.checkpoint_rows(x.cuda())
    dW, _ = ops.grad_weight_rows_q8(q8, dz.cuda())
    v = ops.restore_rows(q8).double().cpu()
    within(dW, dz.double().t() @ v, 44 * E * (dz.double().abs().t() @ v.abs()) + 2.0 ** -149, "dW")
    x[7, 70] = math.nan
    dW, _ = ops.grad_weight_rows_q8(ops.checkpoint_rows(x.cuda()), dz.cuda())
    assert dW[:, 64:96].isnan().all() and dW[:, :64].isfinite().all()


def test_grad_weight_rows_q8_of_many_elements():
    """dW of more elements than one launch has threads for at eight an element.  Three rows: every product is exact and a sum
    of three 32-bit values is off by at most two roundings of the largest partial sum."""
    from mmb_hip import ops
    M, N, K = 3, 23201, 23200
    g = torch.Generator(device="cuda").manual_seed(1)
    q8 = ops.checkpoint_rows(torch.randn(M, K, generator=g, device="cuda"))
    dz = torch.randn(M, N, generator=g, device="cuda")
    dW, db = ops.grad_weight_rows_q8(q8, dz)
    x = ops.restore_rows(q8)
    for lo in range(0, N, 4000):
        z = dz[:, lo:lo + 4000].double()
        tol = 3 * E * (z.abs().t() @ x.double().abs())
        assert bool(((dW[lo:lo + 4000].double() - z.t() @ x.double()).abs() <= tol).all()), lo
    assert bool(((db.double() - dz.double().sum(0)).abs() <= 3 * E * dz.double().abs().sum(0)).all())


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """One conditional attention layer as a training step runs it: project, norm and rotate q and k, attend, project; the
    inputs of the projections are kept as 8-bit checkpoints and the weight gradients come from those."""

    def __init__(self, B, Nq, Nk, d, nh, nkv, D, seed):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.B, self.nh, self.nkv, self.D = B, nh, nkv, D
        self.x, self.c = rnd(B * Nq, d), rnd(B * Nk, d)
        self.Wq, self.Wkv, self.Wo = rnd(nh * D, d) / d ** 0.5, rnd(2 * nkv * D, d) / d ** 0.5, rnd(d, nh * D) / (nh * D) ** 0.5
        self.wq, self.wk = 1 + 0.2 * rnd(D), 1 + 0.2 * rnd(D)
        self.px, self.pc = rnd(B * Nq, 2), rnd(B * Nk, 2)
        self.freq = torch.rand(D // 2, generator=g)
        self.mq, self.mk = slots(B, Nq, g), slots(B, Nk, g)
        self.dy = rnd(B * Nq, d)

    def cuda(self):
        from mmb_hip import ops
        for n, t in list(vars(self).items()):
            if torch.is_tensor(t):
                setattr(self, n, t.cuda())
        self.mq, self.mk = ops.mask_prepare(self.mq), ops.mask_prepare(self.mk)
        return self

    def step(self):
        from mmb_hip import ops
        lin = lambda x, W: ops.linear_cat([(x, ops.SEG_ROW)], W, None, 1)  # noqa: E731
        nk = self.nkv * self.D
        q0, kv = lin(self.x, self.Wq), lin(self.c, self.Wkv)
        cx, cc = ops.checkpoint_rows(self.x), ops.checkpoint_rows(self.c)
        q = ops.head_norm_rotate_fwd(q0, self.nh, self.wq, pos=self.px, freq=self.freq)
        k = ops.head_norm_rotate_fwd(kv[:, :nk], self.nkv, self.wk, pos=self.pc, freq=self.freq)
        kw = dict(mq=self.mq, mk=self.mk)
        a, lse = ops.cross_attention_fwd(q, k, kv[:, nk:], self.B, self.nh, self.nkv, want_lse=True, **kw)
        ca = ops.checkpoint_rows(a)
        y = lin(a, self.Wo)
        da = lin(self.dy, self.Wo.t().contiguous())
        dWo, _ = ops.grad_weight_rows_q8(ca, self.dy)
        dkv = torch.empty_like(kv)
        dq, dk, _ = ops.cross_attention_bwd(q, k, kv[:, nk:], a, da, lse, self.B, self.nh, self.nkv, dv=dkv[:, nk:], **kw)
        dq0, dwq, _ = ops.head_norm_rotate_bwd(q0, dq, self.nh, self.wq, pos=self.px, freq=self.freq)
        _, dwk, _ = ops.head_norm_rotate_bwd(kv[:, :nk], dk, self.nkv, self.wk, pos=self.pc, freq=self.freq, dx=dkv[:, :nk])
        dWq, _ = ops.grad_weight_rows_q8(cx, dq0)
        dWkv, _ = ops.grad_weight_rows_q8(cc, dkv)
        dx, dc = lin(dq0, self.Wq.t().contiguous()), lin(dkv, self.Wkv.t().contiguous())
        return {"y": y, "dx": dx, "dc": dc, "dWq": dWq, "dWkv": dWkv, "dWo": dWo, "dwq": dwq, "dwk": dwk}


def ref_layer(L):
    """The same in 64 bits through autograd, the weight gradients from the 64-bit dZ and the checkpointed inputs."""
    D, B = L.D, L.B
    t = {n: getattr(L, n).double().requires_grad_(True) for n in ("x", "c", "Wq", "Wkv", "Wo", "wq", "wk")}
    nk = L.nkv * D

    def heads(z, w, pos, h):
        z = z.view(z.shape[0], h, D)
        z = z * (z.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        P = D // 2
        ang = pos.double().repeat_interleave(P // 2, 1) * L.freq.double()
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        a, b = z[..., :P], z[..., P:]
        return torch.cat([a * c - b * s, a * s + b * c], -1).view(B, -1, h, D).transpose(1, 2)

    q0, kv = t["x"] @ t["Wq"].t(), t["c"] @ t["Wkv"].t()
    q0.retain_grad()
    kv.retain_grad()
    q, k = heads(q0, t["wq"], L.px, L.nh), heads(kv[:, :nk], t["wk"], L.pc, L.nkv).repeat_interleave(L.nh // L.nkv, 1)
    v = kv[:, nk:].view(B, -1, L.nkv, D).transpose(1, 2).repeat_interleave(L.nh // L.nkv, 1)
    ok = ((L.mq != 0)[:, :, None] & (L.mk != 0)[:, None, :])[:, None]
    s = (D ** -0.5 * q @ k.transpose(2, 3)).masked_fill(~ok, -1e30)
    p = torch.softmax(s, -1) * ok
    a = (p @ v).transpose(1, 2).reshape(L.x.shape[0], -1)
    y = a @ t["Wo"].t()
    (y * L.dy.double()).sum().backward()
    hat = lambda x: ref_codes(x.detach().float())[2]  # noqa: E731
    return {"y": y.detach(), "dx": t["x"].grad, "dc": t["c"].grad, "dWq": q0.grad.t() @ hat(t["x"]), "dWkv": kv.grad.t() @ hat(t["c"]),
            "dWo": L.dy.double().t() @ hat(a), "dwq": t["wq"].grad, "dwk": t["wk"].grad}


@pytest.mark.parametrize("B,Nq,Nk,d,nh,nkv,D", [(3, 50, 70, 64, 4, 2, 16), (2, 1, 150, 64, 4, 4, 16), (2, 130, 40, 128, 4, 1, 32)])
def test_layer_of_all_operators(B, Nq, Nk, d, nh, nkv, D):
    """2^-15 of the largest entry: some twenty 32-bit stages, each off by a few hundred e at these sizes -- but dWo, whose
    checkpoint of the attention's output may land on the other side of a code's border: half the rows by one step is the most
    (a step is 1/64 of its block's largest value at most)."""
    L = Layer(B, Nq, Nk, d, nh, nkv, D, B + Nq)
    want = ref_layer(L)
    got = L.cuda().step()
    for n in want:
        w = want[n]
        tol = 2.0 ** -15 * float(w.abs().max())
        if n == "dWo":
            tol += float(L.dy.abs().double().sum(0).max()) * 2.0 ** -7 * 4 * 2.0 ** -6
        within(got[n], w, torch.full_like(w, tol + 1e-12), n)


def test_layer_captured_and_replayed():
    """Captured into a graph on another stream and replayed with new inputs, eager work between: every replay has the eager
    run's bits; two graphs of the same calls share nothing."""
    L, L2 = Layer(3, 50, 600, 64, 4, 2, 16, 7).cuda(), Layer(3, 50, 600, 64, 4, 2, 16, 8).cuda()
    eager = [{n: t.clone() for n, t in l.step().items()} for l in (L, L2)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(st):
        L.step()
        st.synchronize()
        for l in (L, L2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                res = l.step()
            graphs.append((gr, res))
    torch.cuda.synchronize()
    for turn in range(4):
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i][0].replay()
        L.step()                                                # eager work between the replays
        torch.cuda.synchronize()
        for i in (0, 1):
            for n, t in graphs[i][1].items():
                assert torch.equal(t, eager[i][n]), (turn, i, n)
    x = L.x.clone()
    L.x.copy_(x.flip(0))
    want = {n: t.clone() for n, t in L.step().items()}
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(graphs[0][1][n], want[n]) for n in want) and not torch.equal(want["y"], eager[0]["y"])


def test_two_calls_at_once():
    """Two streams, each with its own workspaces, at the same time."""
    Ls = [Layer(2, 9, 3000, 64, 4, 2, 16, s).cuda() for s in (1, 2)]
    want = [l.step() for l in Ls]
    torch.cuda.synchronize()
    sts = [torch.cuda.Stream() for _ in Ls]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(sts):
            with torch.cuda.stream(st):
                got[i] = Ls[i].step()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[n], w[n]) for n in w)


def test_counts_beyond_32_bits_are_refused():
    from mmb_hip import ops, MMBError
    x, kv = torch.empty(2 ** 32 + 4, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 1, dtype=torch.bfloat16, device="cuda")
    for q, k in ((x, kv), (kv, x)):
        with pytest.raises(MMBError, match="2\\^31"):
            ops.cross_attention_fwd(q, k, k, 1, 1)
    with pytest.raises(MMBError, match="2\\^31"):
        ops.checkpoint_rows(x.view(1, -1))
