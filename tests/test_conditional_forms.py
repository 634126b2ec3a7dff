"""GPU: every form of the conditional operators' kernels -- small clouds with the keys of a head in LDS (16 x 16 tiles in
float, 32 x 32 tiles), eight waves to a tile, keys in two ranges, keys split among waves; the tiles of the weight gradient --
under what the tests of values in test_conditional_ops.py ask of the streaming form alone: masked slots that hold anything,
column slices, values that are not finite, capture and replay, two streams.  References and bounds are those of that file."""
import math

import pytest
import torch

from test_conditional_ops import E, TYPES, check_attention, make, ref_attention, run_attention, within

pytestmark = pytest.mark.gpu

# name: B, Nq, Nk, nh, nkv, D, type.  The small-cloud forms want 256 (cloud, key head) pairs, 8 or 16 queries and a head's keys
# in 53 KB; eight waves 512 workgroups of 256 rows and keys that do not fit; two ranges 256..511 workgroups of 65..128 rows
# and 2560 keys; the split form fewer than 256 workgroups, or 32 rows
FORMS = {
    "tiles of 16, narrow": (300, 33, 40, 2, 1, 16, "f32"),
    "tiles of 16": (256, 70, 90, 2, 2, 32, "f32"),
    "tiles of 16, odd width": (260, 9, 50, 1, 1, 21, "f32"),
    "resident, float": (260, 20, 40, 2, 1, 64, "f32"),
    "resident, bf16": (130, 40, 70, 4, 2, 32, "bf16"),
    "resident, half": (256, 30, 90, 1, 1, 128, "f16"),
    "eight waves": (128, 140, 430, 4, 4, 16, "bf16"),
    "eight waves, float": (128, 131, 200, 4, 4, 40, "f32"),
    "two ranges": (65, 66, 2562, 4, 4, 16, "f16"),
    "split": (3, 20, 900, 2, 1, 64, "f16"),
}
forms = pytest.mark.parametrize("form", list(FORMS))


def args_of(form, masked=True, seed=3):
    B, Nq, Nk, nh, nkv, D, t = FORMS[form]
    return (B, Nq, Nk, nh, nkv, D), TYPES[t], make(B, Nq, Nk, nh, nkv, D, TYPES[t], seed + Nk, masked)


@forms
def test_masked_slots_hold_anything(form):
    (B, Nq, Nk, nh, nkv, D), dt, (q, k, v, do, mq, mk) = args_of(form)
    clean = run_attention(q, k, v, do, mq, mk, B, nh, nkv, 0.3)
    for bad in (math.nan, math.inf, torch.finfo(dt).min):
        dirty = [torch.where(m.reshape(-1, 1) != 0, t, torch.tensor(bad, dtype=dt)) for t, m in ((q, mq), (k, mk), (v, mk), (do, mq))]
        got = run_attention(*dirty, mq, mk, B, nh, nkv, 0.3)
        for n in clean:
            assert torch.equal(got[n], clean[n]), (bad, n)
    gone = (mq == 0).reshape(-1).cuda()
    assert gone.any() and not clean["out"][gone].any() and not clean["dq"][gone].any()
    assert bool((clean["lse"].transpose(1, 2).reshape(B * Nq, nh)[gone] == -math.inf).all())
    gone = (mk == 0).reshape(-1).cuda()
    assert gone.any() and not clean["dk"][gone].any() and not clean["dv"][gone].any()
    assert not clean["out"][Nq:2 * Nq].any()                    # the cloud without a key


@forms
@pytest.mark.parametrize("off", [0, 1])
def test_strides_and_what_lies_around(form, off):
    """Column slices of wider rows, aligned (off 0) and not (off 1): the bits of dense rows, nothing outside is written."""
    from mmb_hip import ops
    (B, Nq, Nk, nh, nkv, D), dt, (q, k, v, do, mq, mk) = args_of(form, seed=5)
    dense = run_attention(q, k, v, do, mq, mk, B, nh, nkv, 0.2)

    def wide(t, fill):
        w = torch.full((t.shape[0] + 3, -(-t.shape[1] // 8) * 8 + 24), 7.0, dtype=dt, device="cuda")
        view = w[1:1 + t.shape[0], 8 + off:8 + off + t.shape[1]]
        if fill:
            view.copy_(t)
        return w, view

    mqi, mki = ops.mask_prepare(mq.cuda()), ops.mask_prepare(mk.cuda())
    qv, kv, vv, gv = (wide(t, True)[1] for t in (q, k, v, do))
    outs = {n: wide(t, False) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    _, lse = ops.cross_attention_fwd(qv, kv, vv, B, nh, nkv, mqi, mki, 0.2, True, outs["out"][1])
    ops.cross_attention_bwd(qv, kv, vv, outs["out"][1], gv, lse, B, nh, nkv, mqi, mki, 0.2, outs["dq"][1], outs["dk"][1], outs["dv"][1])
    assert torch.equal(lse, dense["lse"])
    for n, (w, view) in outs.items():
        assert torch.equal(view, dense[n]), n
        rest = w.clone()
        rest[1:1 + view.shape[0], 8 + off:8 + off + view.shape[1]] = 7.0
        assert bool((rest == 7.0).all()), n


@forms
def test_values_that_are_not_finite(form):
    """A NaN or an infinity in a kept key or value reaches the heads of its own cloud that read it, and nothing else."""
    (B, Nq, Nk, nh, nkv, D), dt, (q, k, v, do, _, _) = args_of(form, masked=False, seed=9)
    base = run_attention(q, k, v, do, None, None, B, nh, nkv, 0.25)
    at, g = min(7, Nk - 1), nh // nkv
    for where, bad in ((k, math.nan), (v, math.nan), (v, math.inf)):
        x = where.clone()
        x[2 * Nk + at, D - 1] = bad                             # cloud 2, key head 0
        got = run_attention(q, x if where is k else k, x if where is v else v, do, None, None, B, nh, nkv, 0.25)
        for n, N, h, spoilt in (("out", Nq, nh, g), ("dq", Nq, nh, g), ("dk", Nk, nkv, 1), ("dv", Nk, nkv, 1)):
            a, b = got[n].view(B, N, h, D).clone(), base[n].view(B, N, h, D).clone()
            if n == "out":
                assert not a[2, :, :g, D - 1].isfinite().any()
            a[2, :, :spoilt] = b[2, :, :spoilt] = 0
            assert torch.equal(a, b), (n, bad)


def step_of(form, seed):
    from mmb_hip import ops
    (B, Nq, Nk, nh, nkv, D), dt, (q, k, v, do, mq, mk) = args_of(form, seed=seed)
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    kw = dict(nheads_kv=nkv, mq=ops.mask_prepare(mq.cuda()), mk=ops.mask_prepare(mk.cuda()), scale=0.25)

    def step():
        out, lse = ops.cross_attention_fwd(q, k, v, B, nh, want_lse=True, **kw)
        return (out, lse) + ops.cross_attention_bwd(q, k, v, out, do, lse, B, nh, **kw)

    return step, q


@forms
def test_captured_and_replayed(form):
    """Two graphs captured on another stream, replayed with eager work between and with new inputs: the eager call's bits."""
    steps = [step_of(form, s) for s in (21, 22)]
    eager = [[t.clone() for t in s()] for s, _ in steps]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(st):
        steps[0][0]()
        st.synchronize()
        for s, _ in steps:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                res = s()
            graphs.append((gr, res))
    torch.cuda.synchronize()
    for turn in range(3):
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i][0].replay()
        steps[0][0]()
        torch.cuda.synchronize()
        for (_, res), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(res, want)), turn
    steps[0][1].copy_(steps[0][1].flip(0))
    want = [t.clone() for t in steps[0][0]()]
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want)) and not torch.equal(want[0], eager[0][0])


@forms
def test_two_streams_at_once(form):
    steps = [step_of(form, s)[0] for s in (31, 32)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    sts, got = [torch.cuda.Stream() for _ in steps], [None, None]
    for _ in range(3):
        for i, st in enumerate(sts):
            with torch.cuda.stream(st):
                got[i] = steps[i]()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("D", [32, 64])
def test_eight_waves_with_several_row_tiles(D, masked, dtype):
    """256 pairs of 300 rows each: two tiles of 256 rows a head, the second one partly filled; too many keys for LDS."""
    B, Nq, Nk, nh = 64, 300, 430, 4
    args = make(B, Nq, Nk, nh, nh, D, TYPES[dtype], D, masked)
    scale = 1.0 / math.sqrt(D)
    check_attention(run_attention(*args, B, nh, nh, scale), ref_attention(*args[:4], B, nh, nh, *args[4:], scale, TYPES[dtype]))


# rows of a head's group, keys: the streaming form on one, two and four waves a workgroup, delta from the row's own p (at most
# 32 keys) and from a launch of its own
SMALL = [(4, 21, 8, 8, 4), (3, 9, 20, 2, 2), (3, 9, 60, 2, 1), (2, 30, 32, 3, 3), (5, 2, 33, 4, 2), (2, 1, 1, 2, 1), (2, 70, 30, 2, 1), (2, 7, 130, 3, 1)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [1, 20, 24, 32, 33, 40, 63, 64, 65, 72, 100, 127, 128])
def test_every_instance_of_the_streaming_form(D, dtype):
    """All head widths (padded to 32, 64, 128; in chunks and element by element) at every number of waves, masked and not.  The
    bounds' sum of first-order errors is widened by 2^-9: two roundings at their worst are 2u + u^2 off, not 2u."""
    dt = TYPES[dtype]
    for i, (B, Nq, Nk, nh, nkv) in enumerate(SMALL):
        print(D, dtype, (B, Nq, Nk, nh, nkv), flush=True)
        args = make(B, Nq, Nk, nh, nkv, D, dt, 100 * i + D, bool(i % 2))
        scale = 1.0 / math.sqrt(D)
        ref = ref_attention(*args[:4], B, nh, nkv, *args[4:], scale, dt)
        check_attention(run_attention(*args, B, nh, nkv, scale), {n: (v, t * (1 + 2.0 ** -9)) for n, (v, t) in ref.items()})


# M, K, N: tiles of 256 x 256 and of 128 x 256, rows of dZ loaded in chunks (N a multiple of 8); ranges of several steps
GRADS = [(700, 264, 248), (2000, 1024, 1000), (515, 320, 64), (900, 320, 320), (65, 256, 256), (31, 136, 136), (3000, 130, 520)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", GRADS)
def test_weight_gradient_tiles(M, K, N, dtype):
    """Values, and column slices beside other columns; the bounds of test_grad_weight_rows_q8."""
    from mmb_hip import ops
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M + K + N)
    q8 = ops.checkpoint_rows((torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).cuda())
    dz = torch.randn(M, N, generator=g).to(dt)
    x, z = ops.restore_rows(q8).double().cpu(), dz.double()
    dW, db = ops.grad_weight_rows_q8(q8, dz.cuda())
    within(dW, z.t() @ x, (M + 4) * E * (z.abs().t() @ x.abs()) + 1e-30, "dW")
    within(db, z.sum(0), (M + 4) * E * z.abs().sum(0) + 1e-30, "db")
    again = ops.grad_weight_rows_q8(q8, dz.cuda())
    assert torch.equal(again[0], dW) and torch.equal(again[1], db)
    wide, zw = torch.ones(N, K + 3, device="cuda"), torch.full((M, N + 16), math.nan, dtype=dt, device="cuda")
    zw[:, 8:8 + N] = dz.cuda()                                  # aligned; the columns around it are not read into any sum
    ops.grad_weight_rows_q8(q8, zw[:, 8:8 + N], dW=wide[:, 2:2 + K], db=db, accumulate=False)
    assert torch.equal(wide[:, 2:2 + K], dW) and bool((wide[:, :2] == 1).all()) and bool((wide[:, 2 + K:] == 1).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(300, 264, 248), (300, 320, 64), (515, 520, 520)])
def test_weight_gradient_tiles_values_that_are_not_finite(M, K, N, dtype):
    """An infinity in a column of dZ reaches that row of dW alone, a checkpoint block of NaN its 32 columns alone -- also
    where the tile's columns past the matrix read a column of it instead."""
    from mmb_hip import ops
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(K)
    x, dz = torch.randn(M, K, generator=g), torch.randn(M, N, generator=g).to(dt)
    base, b0 = ops.grad_weight_rows_q8(ops.checkpoint_rows(x.cuda()), dz.cuda())
    n = (N - 1) // 256 * 256                                    # the first column of the last tile
    bad = dz.clone()
    bad[M // 2, n] = math.inf
    dW, db = ops.grad_weight_rows_q8(ops.checkpoint_rows(x.cuda()), bad.cuda())
    rest = torch.arange(N) != n
    assert not dW[n].isfinite().any() and not db[n].isfinite() and torch.equal(dW[rest], base[rest]) and torch.equal(db[rest], b0[rest])
    x[M - 1, (K - 1) // 256 * 256] = math.nan
    blk = (K - 1) // 256 * 256
    dW, db = ops.grad_weight_rows_q8(ops.checkpoint_rows(x.cuda()), dz.cuda())
    rest = torch.arange(K) // 32 != blk // 32
    assert dW[:, ~rest].isnan().all() and torch.equal(dW[:, rest], base[:, rest]) and torch.equal(db, b0)
