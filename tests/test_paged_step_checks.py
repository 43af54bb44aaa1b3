"""What the operators of a paged serving step refuse, decided on the host before anything is launched; the frequency tables."""
import ctypes as C
import math

import numpy as np
import pytest

from axono_amd import _lib

OK, INVALID, OOM, TYPE, SHAPE, PTR = 0, 1, 2, 3, 4, 7
F16, F32, I32, I64 = 4, 5, 2, 3
P = 0x1000  # an address that the checks look at and nothing reads: every call below ends before a launch


def lib():
    return _lib.load()


def rotary(q=P, qs=128, k=P, ks=64, pos=P, f=P, scale=1.0, inter=0, rd=64, qo=P, ko=P, dt=F16, rows=0, hq=2, hk=1, d=64):
    return lib().axhip_rotary_qk(q, qs, k, ks, pos, f, scale, inter, rd, qo, ko, dt, rows, hq, hk, d, None)


def test_rotary_refusals():
    assert rotary() == OK                            # no rows
    assert rotary(rows=3, hq=0, hk=0) == OK          # no heads
    for bad in (dict(dt=I32), dict(dt=6)):
        assert rotary(rows=1, **bad) == TYPE
    for bad in (dict(rows=-1), dict(hq=-1), dict(d=0), dict(d=60), dict(d=520, qs=1040, ks=520), dict(rd=0), dict(rd=63),
                dict(rd=66), dict(qs=127), dict(ks=63), dict(rows=1 << 31), dict(hq=65000, hk=1000)):
        assert rotary(**{"rows": 1, **bad}) == INVALID, bad
    for bad in (dict(q=None), dict(k=None), dict(pos=None), dict(f=None), dict(qo=None), dict(ko=None), dict(q=P + 1),
                dict(k=P + 1), dict(qo=P + 1), dict(pos=P + 4), dict(f=P + 2), dict(dt=F32, q=P + 2)):
        assert rotary(rows=1, **bad) == PTR, bad
    # an interleaved pair across a boundary of two elements
    assert rotary(rows=1, inter=1, qs=129) == INVALID
    assert rotary(rows=1, inter=1, q=P + 2) == INVALID


def append(dt=F16, wd=F32, norm=1, pos=P, axes=1, rd=64, inter=0, h=0, w=0, cd=F16, T=1, B=1, hq=2, hk=1, d=64, mp=1, n=1, qs=256, ks=256,
           vs=256, **p):
    g = {**dict(q=P, k=P, v=P, qw=P, kw=P, f=P, cu=P, st=P, tb=P, qo=P, kp=P, vp=P), **p}
    return lib().axhip_rotary_append_paged(g["q"], qs, g["k"], ks, g["v"], vs, dt, g["qw"], g["kw"], wd, 1e-6, norm, pos, axes, g["f"], 1.0,
                                           inter, rd, h, w, g["cu"], g["st"], g["tb"], g["qo"], g["kp"], g["vp"], cd, T, B, hq, hk, d, mp,
                                           n, None)


def test_append_refusals():
    assert append(T=0) == OK and append(B=0) == OK
    for bad in (dict(dt=I32), dict(cd=I64), dict(wd=I32)):
        assert append(**bad) == TYPE, bad
    for bad in (dict(T=-1), dict(B=-1), dict(hq=0), dict(hk=0), dict(mp=0), dict(n=0), dict(d=60), dict(d=520), dict(rd=65), dict(rd=0),
                dict(rd=128), dict(axes=2), dict(axes=3, pos=None), dict(h=-1), dict(w=65), dict(qs=127), dict(ks=63), dict(vs=63),
                dict(hq=40000, qs=1 << 30)):
        assert append(**bad) == INVALID, bad
    for name in ("q", "k", "v", "f", "cu", "st", "tb", "qo", "kp", "vp"):
        assert append(**{name: None}) == PTR, name
        assert append(**{name: P + 1}) == PTR, name
    assert append(kp=P + 8) == PTR and append(qw=P + 2) == PTR


def chunk(dt=F16, T=1, B=1, hq=4, hk=2, d=64, mq=1, ml=128, mp=1, n=1, nbytes=1 << 40, **p):
    g = {**dict(q=P, k=P, v=P, tb=P, cu=P, st=P, out=P, ws=P), **p}
    return lib().axhip_chunk_attention_paged(g["q"], g["k"], g["v"], g["tb"], g["cu"], g["st"], g["out"], g["ws"], nbytes, dt, T, B, hq, hk,
                                             d, mq, ml, mp, n, None)


def test_chunk_attention_refusals():
    assert chunk(T=0) == OK and chunk(B=0) == OK and chunk(mq=0) == OK
    assert chunk(dt=I32) == TYPE
    assert chunk(hq=3) == SHAPE
    for bad in (dict(T=-1), dict(B=-1), dict(hq=0), dict(hk=0), dict(d=96), dict(d=32), dict(mq=-1), dict(ml=-1), dict(mp=0), dict(n=0),
                dict(ml=129), dict(T=1 << 29, hq=8), dict(B=(1 << 20) + 1), dict(hk=2000, hq=2000)):
        assert chunk(**bad) == INVALID, bad
    for name in ("q", "k", "v", "tb", "cu", "st", "out"):
        assert chunk(**{name: None}) == PTR, name
        assert chunk(**{name: P + 2}) == PTR, name
    big = dict(ml=4096, mp=32)
    assert chunk(ws=None, **big) == PTR and chunk(ws=P + 8, **big) == PTR
    need = lib().axhip_chunk_attention_paged_workspace_bytes(F16, 1, 1, 4, 2, 64, 1, 4096)
    assert need > 0 and chunk(nbytes=need - 1, **big) == OOM


def test_chunk_attention_workspace():
    size = lib().axhip_chunk_attention_paged_workspace_bytes
    assert size(F16, 5, 2, 4, 2, 64, 5, 256) == 0                  # too few keys to cut
    assert size(F16, 5, 2, 4, 3, 64, 5, 4096) == 0                 # refused sizes need none
    assert size(F16, 65536, 16, 16, 8, 128, 4096, 4096) < 160 << 20
    assert size(F32, 4096, 64, 64, 8, 256, 1, 131072) < 320 << 20


def logits(dt=F32, ls=100, os=100, ht=I32, hr=10, hs=1, H=10, bc=1, als=4, rows=0, V=100, **p):
    g = {**dict(x=P, h=P, hl=P, pl=P, r=P, pr=P, f=P, bi=P, bv=P, al=P, out=P + 4096), **p}
    return lib().axhip_logits_process(g["x"], ls, dt, g["h"], ht, hr, hs, H, g["hl"], g["pl"], g["r"], g["pr"], g["f"], g["bi"], g["bv"], bc,
                                      g["al"], als, g["out"], os, rows, V, None)


def test_logits_refusals():
    assert logits() == OK and logits(rows=1, V=0) == OK
    for bad in (dict(dt=I32), dict(ht=F32)):
        assert logits(rows=1, **bad) == TYPE, bad
    for bad in (dict(rows=-1), dict(rows=70000), dict(V=-1), dict(H=-1), dict(bc=-1), dict(ls=99), dict(os=99), dict(hr=-1), dict(hs=-1),
                dict(als=3), dict(out=P, os=128)):
        assert logits(**{"rows": 1, **bad}) == INVALID, bad
    for bad in (dict(x=None), dict(out=None), dict(bi=None), dict(bv=None), dict(x=P + 2), dict(h=P + 2), dict(hl=P + 1), dict(al=P + 1),
                dict(r=P + 2), dict(ht=I64, h=P + 4)):
        assert logits(rows=1, **bad) == PTR, bad


# ---- frequency tables ----------------------------------------------------------------------------------------------------
def inv_freq(kind, theta, rd, factor=1.0, trained=0, fast=32.0, slow=1.0):
    f, s = np.full(rd // 2, -1, np.float32), C.c_float(-1)
    rc = lib().axhip_rotary_inv_freq(kind, theta, rd, factor, trained, fast, slow, f.ctypes.data, C.byref(s))
    return rc, f, s.value


@pytest.mark.parametrize("rd", [2, 20, 128, 512])
@pytest.mark.parametrize("theta", [1e4, 5e5])
def test_frequency_tables(rd, theta):
    i = np.arange(0, rd, 2, dtype=np.float64) / rd
    plain = theta ** -i
    near = dict(rtol=2.0 ** -24 * 1.01)     # one rounding to fp32 of a value good to a few 2^-53
    rc, f, s = inv_freq(0, theta, rd)
    assert (rc, s) == (OK, 1.0)
    np.testing.assert_allclose(f, plain, **near)
    rc, f, s = inv_freq(1, theta, rd, 8.0)
    assert (rc, s) == (OK, 1.0)
    np.testing.assert_allclose(f, plain / 8, **near)
    rc, f, s = inv_freq(2, theta, rd, 4.0)
    assert (rc, s) == (OK, 1.0)
    np.testing.assert_allclose(f, (theta * 4.0 ** (rd / (rd - 2)) if rd > 2 else theta) ** -i, **near)
    if rd > 2:                              # the slowest pair is slowed by the factor, the fastest not at all
        np.testing.assert_allclose([f[0], f[-1]], [1.0, plain[-1] / 4], **near)
    rc, f, s = inv_freq(3, theta, rd, 16.0, 4096, 32.0, 1.0)
    assert rc == OK and abs(s - (0.1 * math.log(16.0) + 1)) < 2.0 ** -23
    k = np.clip((4096 * plain / (2 * np.pi) - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, plain * k + plain / 16 * (1 - k), **near)
    assert inv_freq(3, theta, rd, 0.5, 4096)[2] == 1.0


def test_frequency_table_refusals():
    for bad in ((4, 1e4, 64), (-1, 1e4, 64), (0, 0.0, 64), (0, float("nan"), 64), (0, 1e4, 514), (1, 1e4, 64, 0.0), (3, 1e4, 64, 2.0, 0),
                (3, 1e4, 64, 2.0, 100, 1.0, 1.0)):
        assert inv_freq(*bad)[0] == INVALID, bad
    assert lib().axhip_rotary_inv_freq(0, 1e4, 63, 1.0, 0, 0.0, 0.0, P, None) == INVALID
    assert lib().axhip_rotary_inv_freq(0, 1e4, 64, 1.0, 0, 0.0, 0.0, None, None) == PTR


def test_host_tensors_are_refused():
    from axono_amd import Status, Tensor, libaxono as L
    from axono_amd.device import AxhipError

    def host(shape, t=np.float32):
        return Tensor.from_numpy_ref(np.zeros(shape, t))

    f, i32 = host(32), np.int32
    pools = (host((2, 1, 128, 64), np.float16),) * 2
    ragged = (host(2, i32), host(1, i32))
    for call in (lambda: L.rotary_qk(host((3, 2, 64)), None, host(3, np.int64), f),
                 lambda: L.rotary_append_paged(host((3, 256)), 2, f, *ragged, *pools, host((1, 2), i32)),
                 lambda: L.chunk_attention_paged(host((3, 2, 64), np.float16), *pools, host((1, 2), i32), *ragged, 3, 128),
                 lambda: L.logits_process(host((2, 100)))):
        with pytest.raises(AxhipError) as e:
            call()
        assert e.value.code == Status.DEVICE_MISMATCH
    table, scale = L.rotary_inv_freq(64, 1e4, "linear", factor=2.0, device="cpu")
    assert scale == 1.0 and table.shape == [32] and abs(float(table.to_numpy()[0]) - 0.5) < 1e-7


def test_sizes_that_no_launch_takes_are_refused():
    # in place with gaps between the rows: a row's result would land on rows that are still to be read
    assert rotary(rows=2, qs=192, qo=P) == INVALID and rotary(rows=2, ks=128, qo=P + 4096, ko=P) == INVALID
    assert append(B=(1 << 20) + 1) == INVALID
    assert chunk(T=1 << 20, B=1 << 20, hq=32, hk=32) == INVALID          # 2^25 workgroups
    assert logits(rows=1, bc=16385) == INVALID


def test_a_plain_frequency_table_looks_at_theta_alone():
    """the factor and the turns of the other kinds are not read"""
    want = inv_freq(0, 1e4, 64)
    for rest in ((0.0,), (-3.0, -1, 1.0, 2.0), (float("nan"), 0, float("nan"), float("nan"))):
        rc, f, s = inv_freq(0, 1e4, 64, *rest)
        assert (rc, s) == (OK, 1.0)
        np.testing.assert_array_equal(f, want[1])
    assert inv_freq(1, 1e4, 64, 2.0, -1, 0.0, 0.0)[0] == OK and inv_freq(2, 1e4, 64, 2.0, -1, 0.0, 0.0)[0] == OK
