"""Refusals of the linear-attention and expert operators: the library's argument checks (compiled for the host) and
the Python mirror's, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

from common import ROOT

EINVAL = -1
P = 1 << 20  # an address that no check looks behind


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("cxx") / "liblayer_checks.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "cxx", "layer_checks.cpp")], check=True)
    lib = ctypes.CDLL(so)
    lib.layer_text.restype = ctypes.c_char_p
    vp, i, ll, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
    lib.layer_conv.argtypes, lib.layer_delta.argtypes = [vp], [vp, sz]
    lib.layer_route.argtypes = [vp, i, i, i, i, vp, vp]
    lib.layer_moe.argtypes = [vp, vp, i, ll, vp, vp, i, vp, ll, i, vp, sz, sz]
    return lib


def test_structs_are_packed_as_the_abi_lays_them_out(lib, qw):
    assert [lib.layer_sizeof(i) for i in range(3)] == [qw._CONV.size, qw._DELTA.size, qw._MOE_LAYER.size]


CONV = dict(n_seq=2, n=5, channels=64, taps=4, dtype=0, lens=0, x=P, x_stride=64, w=P * 2, bias=0, state=P * 3, snap=0,
            y=P * 4, y_stride=64)


def conv_args(qw, **change):
    return qw._CONV.pack(*{**CONV, **change}.values())


@pytest.mark.parametrize("change,text", [
    (dict(n_seq=0), "n_seq"), (dict(n=0), "n 0"), (dict(n=-3), "n -3"), (dict(n_seq=70000), "65535"),
    (dict(n_seq=65535, n=65535), "n_seq"), (dict(channels=60), "multiple of 8"), (dict(channels=0), "channels"),
    (dict(taps=1), "taps"), (dict(taps=5), "taps"), (dict(dtype=2), "dtype 2"), (dict(x=0), "null"), (dict(w=0), "null"),
    (dict(state=0), "null"), (dict(y=0), "null"), (dict(x_stride=56), "x_stride 56"), (dict(y_stride=68), "y_stride 68"),
    (dict(x_stride=-64), "x_stride"), (dict(x=P + 8), "aligned"), (dict(state=P * 3 + 4), "aligned"),
    (dict(y=P), "overlap"), (dict(y=P + 64), "overlap"), (dict(x_stride=128, y_stride=128, y=P + 240), "overlap"),
    (dict(x_stride=128, y_stride=128, y=P + 272), "overlap")])
def test_conv_refuses(lib, qw, change, text):
    assert lib.layer_conv(conv_args(qw, **change)) == EINVAL
    assert text in lib.layer_text().decode()


def test_conv_takes_slices_of_one_buffer(lib, qw):
    assert lib.layer_conv(conv_args(qw)) == 0
    assert lib.layer_conv(conv_args(qw, x_stride=128, y_stride=128, y=P + 256)) == 0
    assert lib.layer_conv(conv_args(qw, x_stride=128, y_stride=128, x=P + 256, y=P)) == 0
    assert lib.layer_conv(conv_args(qw, lens=P, bias=P * 5, snap=P * 6)) == 0


DELTA = dict(n_seq=2, n=5, k_heads=2, v_heads=4, key_dim=64, val_dim=128, tiled=0, dtype=1, lens=0, q=P, k=2 * P, v=3 * P,
             q_stride=128, k_stride=128, v_stride=512, a=4 * P, b=5 * P, a_coef=0, dt_bias=0, state=6 * P, snap=0, z=0,
             z_stride=0, gamma=0, out=7 * P, out_stride=512, workspace=0, workspace_bytes=0)


def delta_args(qw, **change):
    return qw._DELTA.pack(*{**DELTA, **change}.values())


@pytest.mark.parametrize("change,text", [
    (dict(n_seq=0), "n_seq"), (dict(n=0), "n 0"), (dict(k_heads=0), "k_heads"), (dict(v_heads=5), "multiple of k_heads"),
    (dict(v_heads=2048), "1024"), (dict(key_dim=96), "key_dim 96"), (dict(val_dim=256), "val_dim 256"),
    (dict(tiled=2), "tiled 2"), (dict(dtype=2), "dtype 2"), (dict(q=0), "null"), (dict(a=0), "null"), (dict(state=0), "null"),
    (dict(out=0), "null"), (dict(a_coef=P), "together"), (dict(dt_bias=P), "together"), (dict(z=8 * P), "together"),
    (dict(gamma=P), "together"), (dict(q_stride=120), "strides q 120"), (dict(v_stride=516), "v 516"),
    (dict(z=8 * P, gamma=P, z_stride=8), "z 8"), (dict(q=P + 2), "aligned"), (dict(state=P + 8), "aligned"),
    (dict(snap=P + 8), "aligned"), (dict(out=3 * P), "overlaps"), (dict(out=P), "overlaps"),
    (dict(z=7 * P, z_stride=512, gamma=P), "overlaps")])
def test_delta_refuses(lib, qw, change, text):
    assert lib.layer_delta(delta_args(qw, **change), 0) == EINVAL
    assert text in lib.layer_text().decode()


def test_delta_workspace_is_checked(lib, qw):
    assert lib.layer_delta(delta_args(qw), 0) == 0
    for ws, size, rc in ((0, 0, EINVAL), (P, 1023, EINVAL), (P + 16, 1024, EINVAL), (0, 1024, EINVAL), (P, 1024, 0)):
        assert lib.layer_delta(delta_args(qw, workspace=ws, workspace_bytes=size), 1024) == rc
    # q, k and v as slices of one buffer's rows, the output another slice
    one = dict(q=P, k=P + 256, v=P + 512, out=P + 1536, q_stride=2048, k_stride=2048, v_stride=2048, out_stride=2048)
    assert lib.layer_delta(delta_args(qw, **one), 0) == 0


@pytest.mark.parametrize("args,text", [
    ((0, 8, 1, 8, 2, P, P), "null"), ((P, 8, 1, 8, 2, 0, P), "null"), ((P, 8, 0, 8, 2, P, P), "n 0"),
    ((P, 7, 1, 8, 2, P, P), "logits_stride 7"), ((P, 2048, 1, 1025, 2, P, P), "n_experts 1025"),
    ((P, 8, 1, 8, 9, P, P), "top_k 9"), ((P, 8, 1, 8, 0, P, P), "top_k 0"), ((P, 128, 1, 128, 65, P, P), "top_k 65")])
def test_route_refuses(lib, args, text):
    assert lib.layer_route(*args) == EINVAL
    assert text in lib.layer_text().decode()
    assert lib.layer_route(P, 8, 3, 8, 8, P, P) == 0


LAYER = dict(n_experts=4, hidden=64, ffn=96, w_gate=P, w_up=2 * P, w_down=3 * P, s_gate=4 * P, s_up=5 * P, s_down=6 * P)
CALL = dict(x=7 * P, dtype=0, x_stride=64, ids=8 * P, weights=9 * P, top_k=2, y=10 * P, y_stride=64, n=3, ws=11 * P,
            bytes=4096, need=4096)


@pytest.mark.parametrize("layer,call,text", [
    (dict(n_experts=0), {}, "n_experts 0"), (dict(n_experts=1025), {}, "1024"), (dict(hidden=48), {}, "hidden 48"),
    (dict(ffn=0), {}, "ffn 0"), (dict(hidden=65536, ffn=65536), {}, "hidden 65536"), (dict(w_up=0), {}, "null"),
    (dict(s_down=0), {}, "null"), (dict(w_down=P + 8), {}, "aligned"), ({}, dict(x=0), "null"), ({}, dict(ids=0), "null"),
    ({}, dict(n=0), "n 0"), ({}, dict(top_k=65), "top_k 65"), ({}, dict(n=1 << 23, top_k=4), "2^24"),
    ({}, dict(dtype=2), "dtype 2"), ({}, dict(x_stride=60), "x_stride 60"), ({}, dict(y_stride=32), "y_stride 32"),
    ({}, dict(x=7 * P + 4), "aligned"), ({}, dict(y=7 * P), "overlap"), ({}, dict(ws=0), "workspace"),
    ({}, dict(bytes=4095), "workspace"), ({}, dict(ws=11 * P + 128), "workspace")])
def test_moe_refuses(lib, qw, layer, call, text):
    packed = qw._MOE_LAYER.pack(*{**LAYER, **layer}.values())
    assert lib.layer_moe(packed, *{**CALL, **call}.values()) == EINVAL
    assert text in lib.layer_text().decode()
    assert lib.layer_moe(qw._MOE_LAYER.pack(*LAYER.values()), *CALL.values()) == 0


def test_workspace_queries_check_their_sizes(qw):
    assert qw.delta_workspace(1, 1, 2, 4, 128, 128, torch.float32) == 0
    assert qw.moe_workspace(8, 64, 96, torch.float32, 5, 2) > 0
    with pytest.raises(qw.QwattnError, match="key_dim 32"):
        qw.delta_workspace(1, 1, 2, 4, 32, 128, torch.float32)
    with pytest.raises(qw.QwattnError, match="hidden 40"):
        qw.moe_workspace(8, 40, 96, torch.float32, 5, 2)


@pytest.fixture
def att(qw):
    """The Python mirror with no context behind it: its own checks come before any call."""
    a = object.__new__(qw.Attention)
    a.lib, a.h, a.device = qw.load_library(), None, 0
    return a


def test_mirror_refuses(att):
    def z(*s, dtype=torch.float32):
        return torch.zeros(s, dtype=dtype)

    x, w, st = z(2, 3, 16), z(16, 4), z(2, 3, 16)
    for kw, text in ((dict(x=z(2, 3, 16, dtype=torch.float16)), "float32 or bfloat16"), (dict(y=z(2, 4, 16)), "y must be"),
                     (dict(w=z(16, 8)[:, ::2]), "w must be"), (dict(state=z(2, 2, 16)), "state must be"),
                     (dict(x=z(2, 16, 3).transpose(1, 2)), "contiguous"), (dict(x=z(3, 2, 16).transpose(0, 1)), "one stride"),
                     (dict(lens=z(2)), "lens must be"), (dict(snap=z(2, 3, 4, 16)), "snap must be"), ({}, "on cuda:0")):
        with pytest.raises(ValueError, match=text):
            att.conv_silu(**{**dict(x=x, w=w, state=st, y=z(2, 3, 16)), **kw})
    base = dict(q=z(1, 3, 2, 64), k=z(1, 3, 2, 64), v=z(1, 3, 4, 64), a=z(1, 3, 4), b=z(1, 3, 4), state=z(1, 4, 64, 64),
                out=z(1, 3, 4, 64))
    for kw, text in ((dict(q=z(1, 3, 1, 64)), "q must be"), (dict(v=z(1, 3, 4, 64, dtype=torch.bfloat16)), "must be"),
                     (dict(a=z(1, 3, 2)), "a must be"), (dict(state=z(1, 4, 64, 128)), "state must be"),
                     (dict(out=z(1, 3, 64, 4).transpose(2, 3)), "contiguous"), (dict(gamma=z(128)), "gamma must be"), ({}, "on cuda:0")):
        with pytest.raises(ValueError, match=text):
            att.delta_rule(**{**base, **kw})
    for kw, text in ((dict(logits=z(3, 8, dtype=torch.bfloat16)), "logits must be"), (dict(ids=z(3, 2)), "ids must be"),
                     (dict(ids=z(4, 2, dtype=torch.int32)), "ids must be"), (dict(weights=z(3, 1)), "weights must be"),
                     ({}, "on cuda:0")):
        with pytest.raises(ValueError, match=text):
            att.moe_route(**{**dict(logits=z(3, 8), ids=z(3, 2, dtype=torch.int32), weights=z(3, 2)), **kw})
    i8 = dict(dtype=torch.int8)
    up, down = (z(4, 96, 64, **i8), z(4, 96, 2)), (z(4, 64, 96, **i8), z(4, 64, 3))
    call = dict(x=z(3, 64), ids=z(3, 2, dtype=torch.int32), weights=z(3, 2), gate=up, up=up, down=down, y=z(3, 64))
    for kw, text in ((dict(down=up), "down must be"), (dict(up=(up[0], z(4, 96, 3))), "up's scales"),
                     (dict(x=z(3, 32)), "x must be"), (dict(y=z(3, 64, dtype=torch.bfloat16)), "y must be"),
                     (dict(ids=z(3, 2, dtype=torch.int64)), "ids must be"), ({}, "on cuda:0")):
        with pytest.raises(ValueError, match=text):
            att.moe(**{**call, **kw})


def test_sizes_beyond_a_launch_are_refused(lib, qw):
    """Fewer than 2^32 threads in a launch's x: 4,096 a (sequence, value head), 32 a row and head of the gated norm, 64 a
    row of the router in workgroups of four rows."""
    big = dict(k_heads=16, v_heads=32, q_stride=1024, k_stride=1024, v_stride=4096, out_stride=4096, n=1)
    far = {name: (i + 1) << 44 for i, name in enumerate(("q", "k", "v", "z", "out"))}  # apart at any of these sizes
    plain = {**big, **far, "z": 0}
    gated = {**big, **far, "gamma": P, "z_stride": 4096}
    assert 4096 * 32767 * 32 < 2**32 <= 4096 * 32768 * 32
    assert lib.layer_delta(delta_args(qw, **{**plain, "n_seq": 32767}), 0) == 0
    assert lib.layer_delta(delta_args(qw, **{**plain, "n_seq": 32768}), 0) == EINVAL
    assert "2^20" in lib.layer_text().decode()
    n = 2**27 // 32
    assert lib.layer_delta(delta_args(qw, **{**gated, "n_seq": 1, "n": n - 1}), 0) == 0
    assert lib.layer_delta(delta_args(qw, **{**gated, "n_seq": 1, "n": n}), 0) == EINVAL
    assert "2^27" in lib.layer_text().decode()
    assert lib.layer_delta(delta_args(qw, **{**plain, "n_seq": 1, "n": n}), 0) == 0
    most = 2**26 - 5
    assert (most + 3) // 4 * 256 < 2**32
    assert lib.layer_route(P, 8, most, 8, 8, P, P) == 0
    assert lib.layer_route(P, 8, most + 1, 8, 8, P, P) == EINVAL
    assert "2^26" in lib.layer_text().decode()


def test_rows_beyond_32_bit_sums_are_refused(lib, qw):
    """The launchers count tiles (of 16 tokens, doubled while there are more than a grid's y dimension takes) and chunks
    by sums of n and less than a tile: up to the limit they stay below 2^31."""
    most, tile = 2**31 - 2**16, 16
    while (most + tile - 1) // tile > 65535:
        tile *= 2
    assert most + tile - 1 < 2**31
    far = dict(channels=8, dtype=1, x=1 << 44, y=2 << 44, x_stride=8, y_stride=8, n_seq=1)
    assert lib.layer_conv(conv_args(qw, **{**far, "n": most})) == 0
    for n_seq, n in ((1, most + 1), (1, 2**31 - 20001), (1, 2**31 - 1), (2, 2**30 - 2**15 + 1), (65535, 32768)):
        assert lib.layer_conv(conv_args(qw, **{**far, "n_seq": n_seq, "n": n})) == EINVAL
        assert "2^31 - 2^16" in lib.layer_text().decode()
    apart = {name: (i + 1) << 50 for i, name in enumerate(("q", "k", "v", "out"))}
    assert lib.layer_delta(delta_args(qw, **{**apart, "n_seq": 1, "n": most}), 0) == 0
    assert lib.layer_delta(delta_args(qw, **{**apart, "n_seq": 1, "n": most + 1}), 0) == EINVAL
    assert "2^31 - 2^16" in lib.layer_text().decode()


def test_strides_beyond_64_bit_addresses_are_refused(lib, qw):
    """Rows that would span more than 2^59 elements: their byte addresses, and the check for overlaps, stay within 64 bits."""
    rows = 2**31 - 2**16
    most = 2**59 // rows // 8 * 8
    assert rows * most * 4 + 2**57 < 2**63 <= rows * 2**40 * 4
    far = dict(n_seq=1, n=rows, channels=8, x=1 << 44, y=(1 << 44) + 64)
    assert lib.layer_conv(conv_args(qw, **{**CONV, **far, "x_stride": most, "y_stride": most})) == 0  # slices of one buffer
    assert lib.layer_conv(conv_args(qw, **{**CONV, **far, "x_stride": most, "y_stride": most + 8})) == EINVAL
    assert lib.layer_conv(conv_args(qw, **{**CONV, **far, "x_stride": 2**40, "y_stride": 2**40})) == EINVAL
    assert "2^59" in lib.layer_text().decode()
    one = dict(n_seq=1, n=rows, q=1 << 50, k=1 << 51, v=1 << 52, out=1 << 44)  # out ends below the others
    assert lib.layer_delta(delta_args(qw, **{**one, "q_stride": most}), 0) == 0
    for name in ("q", "k", "v", "out"):
        assert lib.layer_delta(delta_args(qw, **{**one, name + "_stride": most + 8}), 0) == EINVAL
        assert "2^59" in lib.layer_text().decode()
    n, layer = 2**22, qw._MOE_LAYER.pack(*LAYER.values())
    for stride, rc in ((2**37, 0), (2**37 + 8, EINVAL), (2**40, EINVAL)):
        call = {**CALL, "n": n, "x": 1 << 50, "y": (1 << 50) + 256, "x_stride": stride, "y_stride": stride}
        assert lib.layer_moe(layer, *call.values()) == rc


def test_a_workspace_serves_every_smaller_call(qw):
    """A program asks once, at its largest: the bytes for (n_seq, n) suffice for any fewer sequences and tokens, for the
    delta rule with z also without, for the experts at any smaller n."""
    lengths = [1, 17, 19, 22, 40, 49, 64, 65, 101, 128, 333, 4096]
    for heads in ((16, 32, 128, 128), (1, 3, 64, 128), (8, 512, 64, 64)):
        for dtype in (torch.float32, torch.bfloat16):
            for gated in (False, True):
                size = {(b, n): qw.delta_workspace(b, n, *heads, dtype, gated) for b in (*range(1, 70), 300) for n in lengths
                        if b * n * heads[1] < 2**27}  # (larger ones are refused with z)
                for (b, n), bytes_ in size.items():
                    assert size[max(1, b - 1 if b < 300 else 69), n] <= bytes_, (heads, dtype, gated, b, n)
                    assert all(size[b, m] <= bytes_ for m in lengths if m < n), (heads, dtype, gated, b, n)
                    assert qw.delta_workspace(b, n, *heads, dtype, False) <= bytes_
    for e, hidden, ffn, k in ((128, 2048, 512, 8), (4, 64, 32, 2), (8, 1024, 352, 2), (1024, 256, 96, 10), (1, 32, 32, 1)):
        for dtype in (torch.float32, torch.bfloat16):
            sizes = [qw.moe_workspace(e, hidden, ffn, dtype, n, k) for n in (*range(1, 600), 2048, 6553, 6554, 20000, 65536, 70000)]
            assert sizes == sorted(sizes)
