"""CPU: what the conditional transformer's entry points refuse -- in the tensor layer, and in the C ABI, where the checks run
on the host before any launch (the addresses handed over here are never touched)."""
import ctypes as C

import pytest
import torch

P = 0x1000                                                     # a 16-byte aligned address


def rc_of(name, *args):
    import mmb_hip
    h = mmb_hip.lib()
    return getattr(h, name)(*args), h.mmb_last_error()


def fwd(**kw):
    a = dict(B=1, Nq=4, Nk=8, nh=2, nkv=1, D=16, dt=0, q=P, q_ld=32, k=P, k_ld=16, v=P, v_ld=16, mq=None, mk=None, scale=0.25, out=P,
             out_ld=32, lse=None, ws=None, n=0, stream=None)
    a.update(kw)
    return rc_of("mmb_cross_attention_fwd", *a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(B=0), b"positive"), (dict(Nq=0), b"positive"), (dict(Nk=0), b"positive"), (dict(Nk=-3), b"positive"),
    (dict(nh=3, nkv=2), b"multiple"), (dict(nkv=0), b"multiple"), (dict(D=0), b"head width"), (dict(D=129), b"head width"),
    (dict(dt=3), b"dtype"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(q=None), b"NULL"), (dict(k=None), b"NULL"), (dict(v=None), b"NULL"),
    (dict(out=None), b"NULL"), (dict(q_ld=31), b"leading"), (dict(k_ld=15), b"leading"), (dict(v_ld=15), b"leading"),
    (dict(out_ld=31), b"leading"), (dict(Nq=1, Nk=100000), b"workspace"), (dict(Nq=1, Nk=100000, ws=P, n=16), b"workspace"),
])
def test_cross_attention_fwd_refuses(kw, word):
    rc, msg = fwd(**kw)
    assert rc == -1 and b"mmb_cross_attention_fwd" in msg and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(lse=None), b"NULL"), (dict(dout=None), b"NULL"), (dict(dk=None), b"NULL"), (dict(dq_ld=31), b"leading"),
    (dict(dv_ld=15), b"leading"), (dict(ws=None), b"workspace"), (dict(n=1 * 2 * 4 * 4 - 1), b"workspace"), (dict(D=200), b"head width"),
])
def test_cross_attention_bwd_refuses(kw, word):
    a = dict(B=1, Nq=4, Nk=8, nh=2, nkv=1, D=16, dt=1, q=P, q_ld=32, k=P, k_ld=16, v=P, v_ld=16, mq=None, mk=None, scale=0.25, out=P,
             out_ld=32, dout=P, dout_ld=32, lse=P, dq=P, dq_ld=32, dk=P, dk_ld=16, dv=P, dv_ld=16, ws=P, n=1 << 20, stream=None)
    a.update(kw)
    rc, msg = rc_of("mmb_cross_attention_bwd", *a.values())
    assert rc == -1 and b"mmb_cross_attention_bwd" in msg and word in msg, msg


def test_workspace_sizes():
    n = C.c_int64(-1)
    assert rc_of("mmb_cross_attention_workspace", 64, 128, 150, 4, 4, 32, 0, 0, C.byref(n))[0] == 0 and n.value == 0
    assert rc_of("mmb_cross_attention_workspace", 1, 1, 100000, 4, 1, 128, 1, 0, C.byref(n))[0] == 0 and n.value > 0
    assert rc_of("mmb_cross_attention_workspace", 3, 5, 7, 4, 1, 8, 1, 1, C.byref(n))[0] == 0 and n.value >= 3 * 4 * 5 * 4
    assert rc_of("mmb_cross_attention_workspace", 3, 5, 7, 4, 3, 8, 1, 1, C.byref(n))[0] == -1
    assert rc_of("mmb_grad_weight_rows_q8_workspace", 1000, 64, 32, C.byref(n))[0] == 0 and n.value >= (64 * 32 + 64) * 4
    assert rc_of("mmb_grad_weight_rows_q8_workspace", 0, 64, 32, C.byref(n))[0] == -1


@pytest.mark.parametrize("kw,word", [
    (dict(M=0), b"positive"), (dict(nh=0), b"positive"), (dict(nh2=-1), b"nheads2"), (dict(D=257, x_ld=10000, y_ld=10000), b"head width"),
    (dict(dt=9), b"dtype"), (dict(x=None), b"NULL"), (dict(y=None), b"NULL"), (dict(x_ld=47), b"leading"), (dict(y_ld=47), b"leading"),
    (dict(eps=0.0), b"eps"), (dict(pairs=9), b"fit"), (dict(pairs=-1), b"fit"), (dict(pos=None), b"need pos"), (dict(freq=None), b"need pos"),
    (dict(axes=3), b"divides"), (dict(axes=0), b"divides"), (dict(pos_ld=1, axes=2), b"divides"), (dict(layout=2), b"layout"),
])
def test_head_norm_refuses(kw, word):
    a = dict(M=3, nh=2, nh2=1, D=16, dt=0, x=P, x_ld=48, w=P, w2=P, eps=1e-6, pos=P, pos_ld=2, axes=2, freq=P, pairs=8, layout=0, y=P,
             y_ld=48, stream=None)
    a.update(kw)
    rc, msg = rc_of("mmb_head_norm_rotate_fwd", *a.values())
    assert rc == -1 and word in msg, msg
    b = list(a.values())
    rc, msg = rc_of("mmb_head_norm_rotate_bwd", *b[:7], P, 48, *b[7:18], None, None, P, None)
    assert rc == -1 and word in msg, msg


def test_head_norm_bwd_refuses():
    a = [3, 2, 1, 16, 0, P, 48, P, 48, P, P, 1e-6, P, 2, 2, P, 8, 0, P, 48, None, None, P, None]
    for i, bad, word in ((7, None, b"dy"), (8, 47, b"dy"), (22, None, b"partials")):
        b = list(a)
        b[i] = bad
        rc, msg = rc_of("mmb_head_norm_rotate_bwd", *b)
        assert rc == -1 and word in msg, msg


@pytest.mark.parametrize("name,args,word", [
    ("mmb_checkpoint_rows", (0, 8, 0, 0, P, 8, P, P, None), b"positive"), ("mmb_checkpoint_rows", (4, 0, 0, 0, P, 8, P, P, None), b"positive"),
    ("mmb_checkpoint_rows", (4, 8, 5, 0, P, 8, P, P, None), b"dtype"), ("mmb_checkpoint_rows", (4, 8, 0, 0, None, 8, P, P, None), b"x is NULL"),
    ("mmb_checkpoint_rows", (4, 8, 0, 0, P, 7, P, P, None), b"leading"), ("mmb_checkpoint_rows", (4, 8, 0, 0, P, 8, None, P, None), b"NULL"),
    ("mmb_checkpoint_rows", (4, 8, 0, 0, P, 8, P + 1, P, None), b"aligned"), ("mmb_restore_rows", (4, 8, 0, P, None, P, 8, None), b"NULL"),
    ("mmb_restore_rows", (4, 8, 0, P, P, None, 8, None), b"NULL"), ("mmb_restore_rows", (4, 8, 0, P, P, P, 7, None), b"leading"),
    ("mmb_restore_rows", (4, 8, 7, P, P, P, 8, None), b"dtype"),
    ("mmb_grad_weight_rows_q8", (4, 8, 0, 0, P, P, P, 8, P, 8, P, 0, P, 1 << 20, None), b"N in"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 0, P, P, None, 8, P, 8, P, 0, P, 1 << 20, None), b"NULL"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 0, P, P, P, 3, P, 8, P, 0, P, 1 << 20, None), b"leading"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 0, P, P, P, 8, P, 7, P, 0, P, 1 << 20, None), b"leading"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 0, P, P, P, 8, P, 8, P, 0, P, 4, None), b"workspace"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 0, P, P, P, 8, P, 8, P, 0, None, 1 << 20, None), b"workspace"),
    ("mmb_grad_weight_rows_q8", (4, 8, 4, 4, P, P, P, 8, P, 8, P, 0, P, 1 << 20, None), b"dtype"),
])
def test_checkpoints_refuse(name, args, word):
    rc, msg = rc_of(name, *args)
    assert rc == -1 and word in msg, msg


def test_tensor_layer_refuses_host_tensors_and_wrong_shapes():
    from mmb_hip import ops, MMBError
    x = torch.zeros(8, 32)
    for call in (lambda: ops.cross_attention_fwd(x, x, x, 2, 2), lambda: ops.cross_attention_bwd(x, x, x, x, x, x, 2, 2),
                 lambda: ops.head_norm_rotate_fwd(x, 2), lambda: ops.head_norm_rotate_bwd(x, x, 2), lambda: ops.checkpoint_rows(x),
                 lambda: ops.restore_rows(ops.Q8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), 20)),
                 lambda: ops.grad_weight_rows_q8(ops.Q8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), 32), x)):
        with pytest.raises(MMBError, match="CPU fallback"):
            call()
    with pytest.raises(MMBError, match="hold rows"):
        ops.Q8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), 33)
    with pytest.raises(MMBError, match="hold rows"):
        ops.Q8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(3, 1, dtype=torch.uint8), 32)
    with pytest.raises(MMBError, match="multiple"):
        ops.cross_attention_fwd(x, x, x, 2, 3, 2)


def test_cross_attention_refuses_outputs_over_inputs():
    at = [0x10000 * (i + 1) for i in range(9)]
    for i in range(3):
        rc, msg = fwd(q=at[0], k=at[1], v=at[2], out=at[i])
        assert rc == -1 and b"an output is the same memory as an input" in msg
    names = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")
    def bwd(over):
        p = dict(zip(names, at), **over)
        return rc_of("mmb_cross_attention_bwd", 1, 4, 8, 2, 1, 16, 1, p["q"], 32, p["k"], 16, p["v"], 16, None, None, 0.25, p["out"], 32,
                     p["dout"], 32, at[8], p["dq"], 32, p["dk"], 16, p["dv"], 16, P, 1 << 20, None)
    for g in names[5:]:
        for i, other in enumerate(names):
            if other != g:
                rc, msg = bwd({g: at[i]})
                assert rc == -1 and b"same memory" in msg, (g, other, msg)


def test_cross_attention_refuses_more_keys_than_its_counters_hold():
    """The kernels count slots in 32 bits and look a step past the last: the largest key counts would wrap around."""
    n, most = C.c_int64(-1), 2 ** 31 - 4097
    for backward in (0, 1):
        assert rc_of("mmb_cross_attention_workspace", 1, 1, most, 1, 1, 1, 2, backward, C.byref(n))[0] == 0 and n.value > 0
    for Nk in (most + 1, 2 ** 31 - 513, 2 ** 31 - 1):
        for backward in (0, 1):
            rc, msg = rc_of("mmb_cross_attention_workspace", 1, 1, Nk, 1, 1, 1, 2, backward, C.byref(n))
            assert rc == -1 and b"Nk must not exceed" in msg, msg
        rc, msg = fwd(Nq=1, Nk=Nk, nh=1, nkv=1, D=1, dt=2, mk=P)
        assert rc == -1 and b"Nk must not exceed" in msg, msg


class Box:
    """Byte addresses of column slices in rows of 256 floats, two of them at the same place."""
    base, ld = 0x100000, 256

    def __call__(self, col, row=0):
        return self.base + 4 * (row * self.ld + col)


def fwd_in_box(**kw):
    """B = 2, Nq = 4, Nk = 8, 2 heads on 1 of 16 floats: q, out 8 rows of 32; k, v 16 rows of 16, all slices of rows of 256"""
    at = Box()
    a = dict(B=2, Nq=4, Nk=8, nh=2, nkv=1, D=16, dt=0, q=at(0), q_ld=256, k=at(64), k_ld=256, v=at(96), v_ld=256, mq=0x10000, mk=0x20000,
             scale=0.25, out=at(128), out_ld=256, lse=0x30000, ws=None, n=0, stream=None)
    a.update(kw)
    return rc_of("mmb_cross_attention_fwd", *a.values())


@pytest.mark.parametrize("kw", [
    dict(out=Box()(16)), dict(out=Box()(31)), dict(out=Box()(0, 1)), dict(out=Box()(0, 7)), dict(out=Box()(240)),
    dict(out=Box()(48)), dict(out=Box()(79, 3)), dict(out=Box()(100)), dict(out=Box()(250, 2)), dict(out=Box()(0), out_ld=512),
    dict(out=Box()(224), out_ld=288), dict(lse=Box()(0, 3)), dict(lse=0x10000), dict(lse=0x2003c), dict(out=0x30000), dict(out=0x10010, out_ld=32),
])
def test_cross_attention_fwd_refuses_partial_overlaps(kw):
    rc, msg = fwd_in_box(**kw)
    assert rc == -1 and b"overlap" in msg, msg


def test_cross_attention_bwd_refuses_partial_overlaps():
    at = Box()
    ok = dict(q=at(0), k=at(32), v=at(48), out=at(64), dout=at(96), lse=0x30000, dq=at(128), dk=at(160), dv=at(176), ws=0x40000)
    def bwd(**kw):
        p = dict(ok, **kw)
        return rc_of("mmb_cross_attention_bwd", 2, 4, 8, 2, 1, 16, 0, p["q"], 256, p["k"], 256, p["v"], 256, 0x10000, 0x20000, 0.25, p["out"],
                     256, p["dout"], 256, p["lse"], p["dq"], 256, p["dk"], 256, p["dv"], 256, p["ws"], 1 << 20, None)
    for kw in (dict(dq=at(100)), dict(dk=at(150)), dict(dv=at(160, 5)), dict(dk=at(8, 2)), dict(dv=at(64)), dict(dq=at(240, 1)),
               dict(ws=0x30000), dict(ws=0x10000), dict(ws=0x20004), dict(ws=at(130, 2)), dict(dq=0x30004), dict(ws=0x30000 + 60)):
        rc, msg = bwd(**kw)
        assert rc == -1 and b"overlap" in msg, (kw, msg)


def test_head_norm_refuses_overlaps():
    """Over x itself (dx over dy or x) is fine, row for row; shifted, at another stride or over the small inputs it is not."""
    ok = dict(M=4, nh=2, nh2=1, D=16, dt=0, x=0x100000, x_ld=64, w=0x10000, w2=0x11000, eps=1e-6, pos=0x12000, pos_ld=2, axes=2, freq=0x13000,
              pairs=8, layout=0, y=0x200000, y_ld=64, stream=None)
    for kw in (dict(y=0x100000, y_ld=48), dict(y=0x100000 + 4), dict(y=0x100000 + 64 * 4), dict(y=0x100000 - 4 * 40), dict(y=0x10020),
               dict(y=0x11000), dict(y=0x12010), dict(y=0x13000)):
        a = dict(ok, **kw)
        rc, msg = rc_of("mmb_head_norm_rotate_fwd", *a.values())
        assert rc == -1 and b"overlap" in msg, (kw, msg)
        for dy in (0x300000, a["y"]):                                # (dx over dy does not excuse dx over x)
            b = list(a.values())
            rc, msg = rc_of("mmb_head_norm_rotate_bwd", *b[:7], dy, a["y_ld"], *b[7:18], None, None, 0x400000, None)
            assert rc == -1 and b"overlap" in msg, (kw, msg)
    b = list(ok.values())
    for dy, dy_ld, d1, d2, part in ((0x200000, 48, None, None, 0x400000), (0x200004, 64, None, None, 0x400000), (0x300000, 64, 0x200000, None, 0x400000),
                                    (0x300000, 64, 0x100010, None, 0x400000), (0x300000, 64, 0x500000, 0x500020, 0x400000),
                                    (0x300000, 64, 0x400000, None, 0x400000), (0x300000, 64, None, None, 0x100000 - 64), (0x300000, 64, 0x10000, None, 0x400000)):
        rc, msg = rc_of("mmb_head_norm_rotate_bwd", *b[:7], dy, dy_ld, *b[7:18], d1, d2, part, None)
        assert rc == -1 and b"overlap" in msg, msg


@pytest.mark.parametrize("name,args", [
    ("mmb_checkpoint_rows", (4, 40, 0, 0, 0x1000, 40, 0x1010, 0x9000, None)), ("mmb_checkpoint_rows", (4, 40, 0, 0, 0x1000, 40, 0x8000, 0x1100, None)),
    ("mmb_checkpoint_rows", (4, 40, 1, 0, 0x1000, 40, 0x8000, 0x8040, None)),
    ("mmb_restore_rows", (4, 40, 0, 0x8000, 0x9000, 0x80f0, 40, None)), ("mmb_restore_rows", (4, 40, 2, 0x8000, 0x9000, 0x8fff, 40, None)),
    ("mmb_grad_weight_rows_q8", (4, 8, 6, 0, 0x1000, 0x2000, 0x3000, 6, 0x3040, 8, None, 0, 0x8000, 1 << 20, None)),
    ("mmb_grad_weight_rows_q8", (4, 8, 6, 0, 0x1000, 0x2000, 0x3000, 6, 0x4000, 8, 0x3000, 0, 0x8000, 1 << 20, None)),
    ("mmb_grad_weight_rows_q8", (4, 8, 6, 0, 0x1000, 0x2000, 0x3000, 6, 0x4000, 8, 0x4010, 0, 0x8000, 1 << 20, None)),
    ("mmb_grad_weight_rows_q8", (4, 8, 6, 0, 0x1000, 0x2000, 0x3000, 6, 0x4000, 8, 0x5000, 0, 0x1040, 1 << 20, None)),
    ("mmb_grad_weight_rows_q8", (4, 8, 6, 0, 0x1000, 0x2000, 0x3000, 6, 0x8010, 8, 0x5000, 0, 0x8000, 1 << 20, None)),
])
def test_checkpoints_refuse_overlaps(name, args):
    rc, msg = rc_of(name, *args)
    assert rc == -1 and b"overlap" in msg, msg


@pytest.mark.parametrize("shape", [  # B, Nq, Nk, nh, nkv, D, dtype: the small-cloud forms, one wave, eight waves
    (1 << 20, 8, 8, 16, 16, 16, 0), (1 << 20, 16, 16, 16, 16, 64, 2), (1 << 22, 1, 8, 64, 64, 1, 1), (1 << 20, 300, 400, 8, 8, 128, 1)])
def test_cross_attention_refuses_more_workgroups_than_a_launch_takes(shape):
    B, Nq, Nk, nh, nkv, D, dt = shape
    far = [(i + 1) << 46 for i in range(9)]
    rc, msg = fwd(B=B, Nq=Nq, Nk=Nk, nh=nh, nkv=nkv, D=D, dt=dt, q=far[0], q_ld=nh * D, k=far[1], k_ld=nkv * D, v=far[2], v_ld=nkv * D, out=far[3],
                  out_ld=nh * D)
    assert rc == -1 and b"workgroups" in msg, msg
    rc, msg = rc_of("mmb_cross_attention_bwd", B, Nq, Nk, nh, nkv, D, dt, far[0], nh * D, far[1], nkv * D, far[2], nkv * D, None, None, 0.25,
                    far[3], nh * D, far[4], nh * D, far[5], far[6], nh * D, far[7], nkv * D, far[8], nkv * D, 3 << 45, 1 << 40, None)
    assert rc == -1 and b"workgroups" in msg, msg


def test_cross_attention_refuses_tiles_beyond_32_bits():
    rc, msg = rc_of("mmb_cross_attention_bwd", 1, 1, 2 ** 31 - 5000, 1024, 1024, 1, 2, 1 << 46, 1024, 1 << 47, 1024, 1 << 48, 1024, None, None,
                    0.25, 1 << 49, 1024, 1 << 50, 1024, 1 << 51, 1 << 52, 1024, 1 << 53, 1024, 1 << 54, 1024, 1 << 55, 1 << 40, None)
    assert rc == -1 and b"workgroups" in msg, msg


def test_workspace_query_refuses_what_the_call_refuses():
    """N and K up to 2^20: beyond, the query's own divisions would run past 32 bits."""
    n = C.c_int64(-1)
    assert rc_of("mmb_grad_weight_rows_q8_workspace", 8, 1 << 20, 1 << 20, C.byref(n))[0] == 0 and n.value == 4 * ((1 << 40) + (1 << 20))
    for N, K in (((1 << 20) + 1, 8), (8, (1 << 20) + 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        rc, msg = rc_of("mmb_grad_weight_rows_q8_workspace", 8, N, K, C.byref(n))
        assert rc == -1 and b"at most 2^20" in msg, msg


def kernels_of(path):
    """Names and resources of the GPU kernels in a library: the metadata notes of the code objects that it carries."""
    import struct
    msgpack = pytest.importorskip("msgpack")
    data = open(path, "rb").read()
    at = data.find(b"\x7fELF\x02\x01\x01\x40")
    while at >= 0:
        if struct.unpack_from("<H", data, at + 18)[0] == 224:       # a GPU's machine number
            table, count = struct.unpack_from("<Q", data, at + 40)[0], struct.unpack_from("<H", data, at + 60)[0]
            for i in range(count):
                section = at + table + 64 * i
                if struct.unpack_from("<I", data, section + 4)[0] == 7:                     # notes
                    note = at + struct.unpack_from("<Q", data, section + 24)[0]
                    name, size, _ = struct.unpack_from("<III", data, note)
                    start = note + 12 + (name + 3) // 4 * 4
                    yield from msgpack.unpackb(data[start:start + size], strict_map_key=False)["amdhsa.kernels"]
        at = data.find(b"\x7fELF\x02\x01\x01\x40", at + 4)


def test_no_kernel_of_the_conditional_operators_spills_registers():
    """The compiler has stored a spilled register under a narrowed exec mask and read it back for all lanes: the reverse of cross
    attention (bfloat16, head widths off the chunk of eight between 33 and 63, two waves, at most 32 keys) then wrote to
    addresses that scratch memory happened to hold.  Without spills there is nothing to misplace."""
    import mmb_hip
    ours = [k for k in kernels_of(mmb_hip.LIB_PATH) if any(n in k[".name"] for n in ("3mmb5xattn", "3mmb8headnorm", "3mmb4ckpt"))]
    assert len(ours) > 100
    assert not [(k[".name"], k[".vgpr_spill_count"]) for k in ours if k[".vgpr_spill_count"]]
