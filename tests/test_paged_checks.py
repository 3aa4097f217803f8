"""Refusals of the paged-attention operators: the library's argument checks (compiled for the host) and the Python
mirror's, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

from common import ROOT

EINVAL = -1
P = 1 << 30  # an address that no check looks behind; the operands lie P apart


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("cxx") / "libpaged_checks.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "cxx", "paged_checks.cpp")], check=True)
    lib = ctypes.CDLL(so)
    lib.paged_text.restype = ctypes.c_char_p
    lib.paged_append.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    lib.paged_attend.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t]
    return lib


@pytest.fixture(scope="module")
def shape(qw):
    return qw.Config(8, 2, 64, 32, 1e7, 1e-6, 1024, 64, 64)


def test_structs_are_packed_as_the_abi_lays_them_out(lib, qw):
    assert [lib.paged_sizeof(0), lib.paged_sizeof(1)] == [qw._PAGED_APPEND.size, qw._PAGED_ATTEND.size]


CACHE = dict(kpool=P, vpool=2 * P, table=3 * P, table_stride=4, n_pages=10, pages=4, page=32)
APPEND = dict(**CACHE, n_seq=2, n=5, dtype=0, n_rope=0, lens=0, pos=4 * P, q=5 * P, q_stride=1024, q_head=128, k=6 * P, v=7 * P,
              k_stride=128, v_stride=128, qn=8 * P, kn=9 * P, rope=0, q_out=10 * P, q_out_stride=512)
ATTEND = dict(**CACHE, n_seq=2, n=5, dtype=1, window=0, sinks=0, scale=0.0, lens=0, pos=4 * P, q=5 * P, q_stride=512, q_head=64,
              gate=6 * P, gate_stride=1024, gate_head=128, out=7 * P, out_stride=512, ws=8 * P, bytes=4096)
POOL = 10 * 32 * 2 * 64 * 2  # bytes of a pool

BAD_CACHE = [(dict(n_seq=0), "n_seq 0"), (dict(n=0), "n 0"), (dict(n=-1), "n -1"), (dict(n_seq=70000), "65535"),
             (dict(n_seq=65535, n=1000), "2^26"), (dict(page=16), "page 16"), (dict(page=96), "page 96"), (dict(page=1 << 17), "page"),
             (dict(n_pages=0), "n_pages 0"), (dict(n_pages=(1 << 30) + 1), "2^31"), (dict(pages=0), "pages 0"), (dict(pages=1 << 22, table_stride=1 << 22), "2^26"),
             (dict(n_seq=65535, n=1, pages=1 << 16, table_stride=1 << 16), "2^36"), (dict(kpool=0), "null"), (dict(vpool=0), "null"), (dict(table=0), "null"), (dict(table_stride=3), "table_stride 3"),
             (dict(kpool=P + 8), "aligned"), (dict(table=3 * P + 2), "aligned"), (dict(vpool=P + POOL - 16), "pools overlap"),
             (dict(pos=0), "pos"), (dict(dtype=2), "dtype 2")]


@pytest.mark.parametrize("change,text", BAD_CACHE + [
    (dict(q_out=0), "together"), (dict(q=0), "together"), (dict(rope=P, n_rope=0), "n_rope 0"), (dict(qn=8 * P + 4), "aligned"),
    (dict(rope=P + 4, n_rope=9), "aligned"), (dict(k=0), "k is null"), (dict(v=0), "v is null"), (dict(k_stride=120), "k's strides 120"),
    (dict(v_stride=132), "v's strides 132"), (dict(q_head=60), "q's strides"), (dict(q_head=68), "q's strides"),
    (dict(q_stride=952), "q's strides 952"), (dict(q=5 * P + 8), "aligned"), (dict(q_out_stride=504), "q_out's strides 504"),
    (dict(q_out=5 * P), "overlaps q"), (dict(q_out=6 * P), "overlaps k"), (dict(k=P + 64), "k overlaps the pools"),
    (dict(q_out=2 * P + POOL - 64), "q_out overlaps the pools"), (dict(q_stride=1 << 60), "2^59")])
def test_append_refuses(lib, qw, shape, change, text):
    assert lib.paged_append(qw._PAGED_APPEND.pack(*{**APPEND, **change}.values()), ctypes.byref(shape)) == EINVAL
    assert text in lib.paged_text().decode()


def test_append_takes(lib, qw, shape):
    for change in ({}, dict(q=0, q_out=0), dict(rope=P, n_rope=1), dict(lens=P), dict(kn=0, qn=0),
                   dict(q_head=64, q_stride=512), dict(q=5 * P, k=5 * P + 2048, v=5 * P + 2560, q_stride=1024, k_stride=1024, v_stride=1024, q_head=64)):
        assert lib.paged_append(qw._PAGED_APPEND.pack(*{**APPEND, **change}.values()), ctypes.byref(shape)) == 0, lib.paged_text()


@pytest.mark.parametrize("change,text", BAD_CACHE + [
    (dict(window=-1), "window -1"), (dict(sinks=-2), "sinks -2"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=0), "q is null"), (dict(out=0), "out is null"), (dict(gate_head=56), "gate's strides"),
    (dict(gate_stride=900), "gate's strides"), (dict(q_stride=504), "q's strides"), (dict(out=5 * P), "overlaps q"),
    (dict(out=6 * P), "overlaps gate"), (dict(out=P), "overlaps the pools"), (dict(out_stride=500), "out's strides"),
    (dict(ws=0), "workspace"), (dict(bytes=4095), "workspace"), (dict(ws=8 * P + 64), "workspace")])
def test_attend_refuses(lib, qw, shape, change, text):
    assert lib.paged_attend(qw._PAGED_ATTEND.pack(*{**ATTEND, **change}.values()), ctypes.byref(shape), 4096) == EINVAL
    assert text in lib.paged_text().decode()


def test_attend_takes(lib, qw, shape):
    for change in ({}, dict(gate=0), dict(window=7, sinks=1 << 30), dict(scale=3.0), dict(q=6 * P + 128, q_head=128, q_stride=1024)):
        assert lib.paged_attend(qw._PAGED_ATTEND.pack(*{**ATTEND, **change}.values()), ctypes.byref(shape), 4096) == 0, lib.paged_text()


@pytest.fixture
def att(qw):
    """The Python mirror with no context behind it: its own checks come before any call."""
    a = object.__new__(qw.Attention)
    a.lib, a.h, a.device, a.NH, a.NKV, a.D, a.R = qw.load_library(), None, 0, 8, 2, 64, 32
    return a


def z(*s, dtype=torch.float32):
    return torch.zeros(s, dtype=dtype)


def test_mirror_refuses(att):
    i32, h = torch.int32, torch.float16
    pools = dict(kpool=z(9, 2, 64 * 64, dtype=h), vpool=z(9, 2, 64 * 64, dtype=h), table=z(2, 3, dtype=i32), pos=z(2, dtype=i32))
    bad_pools = [(dict(kpool=z(9, 2, 64 * 64)), "kpool must be"), (dict(kpool=z(9, 4, 64 * 64, dtype=h)), "kpool must be"),
                 (dict(vpool=z(8, 2, 64 * 64, dtype=h)), "vpool must be"), (dict(kpool=z(9, 2, 65, dtype=h)), "kpool must be"),
                 (dict(table=z(3, 3, dtype=i32)), "table must be"), (dict(table=z(2, 3)), "table must be"),
                 (dict(table=z(3, 2, dtype=i32).t()), "table must be"), (dict(pos=z(3, dtype=i32)), "pos must be"),
                 (dict(pos=z(2)), "pos must be"), (dict(lens=z(1, dtype=i32)), "lens must be")]
    good = dict(k=z(2, 5, 2, 64), v=z(2, 5, 2, 64), **pools, q=z(2, 5, 8, 128)[..., :64], q_out=z(2, 5, 8, 64))
    for kw, text in bad_pools + [
            (dict(k=z(2, 5, 2, 64, dtype=h)), "k must be"), (dict(k=z(2, 5, 2, 32)), "k must be"), (dict(v=z(2, 4, 2, 64)), "v must be"),
            (dict(q=z(2, 5, 8, 64, dtype=torch.bfloat16)), "q must be"), (dict(q=z(2, 5, 8, 128)[..., ::2]), "q: a head"),
            (dict(q=z(2, 6, 8, 64)[:, :5]), "q: a head"), (dict(q_out=z(2, 5, 8, 128)[..., :64]), "contiguous"),
            (dict(qn=z(32)), "qn must be"), (dict(kn=z(64).double()), "kn must be"), (dict(rope=z(9, 16, 3)), "rope must be"),
            (dict(k=z(2, 5, 2, 64)), "must be on cuda:0")]:
        with pytest.raises(ValueError, match=text):
            att.paged_append(**{**good, **kw})
    good = dict(q=z(2, 5, 8, 64), **pools, out=z(2, 5, 8, 64))
    for kw, text in bad_pools + [
            (dict(q=z(2, 5, 8, 64, dtype=h)), "q must be"), (dict(q=z(2, 5, 4, 64)), "q must be"), (dict(out=z(2, 5, 8, 64).bfloat16()), "out must be"),
            (dict(gate=z(2, 5, 8, 32)), "gate must be"), (dict(q=z(2, 5, 8, 64)), "must be on cuda:0")]:
        with pytest.raises(ValueError, match=text):
            att.paged_attend(**{**good, **kw})


def test_entry_points_need_a_context(qw):
    lib = qw.load_library()
    assert lib.qwattn_paged_append(None, None, None) == EINVAL
    assert lib.qwattn_paged_attend(None, None, None) == EINVAL
    assert lib.qwattn_paged_workspace(None, None) == EINVAL


def test_attend_refuses_scales_that_pass_fp32_in_base_2(lib, qw, shape):
    """The kernels take the scale times log2(e): 2^126 is the largest power of two that stays finite."""
    pack = lambda x: qw._PAGED_ATTEND.pack(*{**ATTEND, "scale": x}.values())  # noqa: E731
    assert lib.paged_attend(pack(2.0 ** 126), ctypes.byref(shape), 4096) == 0
    for x in (2.0 ** 126 * (1 + 2.0 ** -23), 2.5e38, 3.3e38):
        assert lib.paged_attend(pack(x), ctypes.byref(shape), 4096) == EINVAL and "scale" in lib.paged_text().decode()


def test_mirror_takes_a_table_of_one_page_at_any_stride(att):
    """(refused only for being on the CPU)"""
    pools = dict(kpool=z(9, 2, 64 * 64, dtype=torch.float16), vpool=z(9, 2, 64 * 64, dtype=torch.float16), pos=z(2, dtype=torch.int32))
    for table in (z(1, 2, dtype=torch.int32).t(), z(2, 6, dtype=torch.int32)[:, ::7], z(2, 1, dtype=torch.int32)):
        assert table.shape == (2, 1)
        with pytest.raises(ValueError, match="must be on cuda:0"):
            att.paged_attend(z(2, 5, 8, 64), table=table, out=z(2, 5, 8, 64), **pools)
