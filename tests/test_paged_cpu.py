"""The paged cache operators' refusals, without a GPU: the C ABI checks its
arguments before any launch, and the Python layer before it reaches the
library."""
import ctypes

import pytest
import torch

from kudahitam import _lib, lloyd_max, ops, rademacher

D128 = (ctypes.c_float * 128)(*([1.0, -1.0] * 64))
C2 = (ctypes.c_float * 2)(-0.07, 0.07)
FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x10002)
OK, INVAL, ALIGN, NOTSUP = _lib.KH_OK, _lib.KH_EINVAL, _lib.KH_EALIGN, _lib.KH_ENOTSUP


def _cache(**kw):
    a = dict(n_pages=4, page_size=16, n_kv_heads=2, head_dim=128)
    a.update({n: 0x10000 for n, _ in _lib.PagedCache._fields_[:8]})
    a.update(kw)
    return _lib.PagedCache(**a)


def _append(cache=None, **kw):
    a = dict(k=FAKE, v=FAKE, dtype=_lib.KH_BF16, n=3, kts=256, khs=128, vts=256, vhs=128,
             slots=FAKE, positions=FAKE, cos=FAKE, sin=FAKE, n_pos=10, rot=128, inter=0, dk=D128,
             dv=D128, c=C2, n_c=2)
    a.update(kw)
    c = cache if cache is not None else _cache()
    return _lib.lib().kh_paged_append(ctypes.byref(c), a["k"], a["v"], a["dtype"], a["n"], a["kts"],
                                      a["khs"], a["vts"], a["vhs"], a["slots"], a["positions"],
                                      a["cos"], a["sin"], a["n_pos"], a["rot"], a["inter"],
                                      a["dk"], a["dv"], a["c"], a["n_c"], None)


BAD_CACHES = [(dict(head_dim=64), INVAL), (dict(page_size=0), INVAL), (dict(n_kv_heads=0), INVAL),
              (dict(n_pages=-1), INVAL), (dict(n_pages=1 << 31), INVAL), (dict(k_res=0), INVAL),
              (dict(v_code=0x10008), ALIGN), (dict(v_norms=0x10004), ALIGN)]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_append_refuses_bad_caches(kw, status):
    assert _append(_cache(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=5), INVAL), (dict(n=-1), INVAL), (dict(k=None), INVAL), (dict(v=None), INVAL),
    (dict(slots=None), INVAL), (dict(k=ctypes.c_void_p(0x10001)), ALIGN),
    (dict(slots=ctypes.c_void_p(0x10004)), ALIGN), (dict(cos=None), INVAL),
    (dict(n_pos=0), INVAL), (dict(rot=0), INVAL), (dict(rot=129), INVAL), (dict(rot=130), INVAL),
    (dict(inter=2), INVAL), (dict(positions=ctypes.c_void_p(0x10004)), ALIGN),
    (dict(dk=(ctypes.c_float * 128)(*([0.5] * 128))), INVAL), (dict(c=None), INVAL),
    (dict(c=(ctypes.c_float * 4)(-0.2, -0.1, 0.1, 0.2), n_c=4), NOTSUP), (dict(n_c=3), INVAL),
    (dict(n=0), OK),
])
def test_append_refuses_bad_arguments(kw, status):
    assert _append(**kw) == status


def _attn(cache=None, **kw):
    a = dict(q=FAKE, dtype=_lib.KH_BF16, B=2, n_q=4, table=FAKE, ts=8, lengths=FAKE, starts=None,
             max_len=100, prefix=0, window=0, cap=0.0, slopes=None, scale=0.1, dk=D128, dv=D128,
             c=C2, n_c=2, ws=FAKE, wb=1 << 40, out=FAKE, lse=None)
    a.update(kw)
    c = cache if cache is not None else _cache()
    return _lib.lib().kh_paged_attn(ctypes.byref(c), a["q"], a["dtype"], a["B"], a["n_q"],
                                    a["table"], a["ts"], a["lengths"], a["starts"], a["max_len"],
                                    a["prefix"], a["window"], a["cap"], a["slopes"], a["scale"],
                                    a["dk"], a["dv"], a["c"], a["n_c"], a["ws"], a["wb"], a["out"],
                                    a["lse"], None)


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_attention_refuses_bad_caches(kw, status):
    assert _attn(_cache(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), INVAL), (dict(B=-1), INVAL), (dict(n_q=0), INVAL), (dict(max_len=-1), INVAL),
    (dict(max_len=1 << 31), INVAL), (dict(prefix=-1), INVAL), (dict(prefix=101), INVAL),
    (dict(window=-1), INVAL), (dict(cap=-1.0), INVAL), (dict(cap=float("inf")), INVAL),
    (dict(scale=float("nan")), INVAL), (dict(ts=6), INVAL), (dict(ts=-1, B=1), INVAL),
    (dict(q=None), INVAL), (dict(out=None), INVAL), (dict(lengths=None), INVAL),
    (dict(table=None), INVAL), (dict(ws=None), INVAL), (dict(wb=16), INVAL),
    (dict(q=ctypes.c_void_p(0x10001)), ALIGN), (dict(lengths=ODD), ALIGN), (dict(table=ODD), ALIGN),
    (dict(starts=ODD), ALIGN), (dict(slopes=ODD), ALIGN), (dict(lse=ODD), ALIGN),
    (dict(ws=ctypes.c_void_p(0x10008)), ALIGN), (dict(n_c=3), INVAL),
    (dict(c=(ctypes.c_float * 4)(-0.2, -0.1, 0.1, 0.2), n_c=4), NOTSUP),
    (dict(B=1 << 30), INVAL), (dict(B=0), OK),
])
def test_attention_refuses_bad_arguments(kw, status):
    assert _attn(**kw) == status


def test_workspace_sizes():
    def f(n_seqs, n_q, heads, D, max_len, prefix=0, window=0, dtype=_lib.KH_BF16):
        return _lib.lib().kh_paged_workspace_bytes(n_seqs, n_q, heads, D, dtype, max_len, prefix,
                                                   window)
    assert f(3, 1, 1, 128, 0) == 0  # nothing can be attended
    assert f(2, 4, 8, 128, 100) >= 2 * 4 * 8 * 130 * 4
    assert f(2, 4, 8, 96, 100) == -1 and f(2, 4, 8, 128, 100, 101) == -1
    assert f(2, 0, 8, 128, 100) == -1 and f(-1, 1, 1, 128, 1) == -1
    assert f(2, 4, 8, 128, 100, dtype=7) == -1
    # a window bounds what a sequence needs; records do not grow without bound
    assert f(64, 1, 8, 128, 100000, 0, 64) < f(64, 1, 8, 128, 100000)
    assert f(64, 4, 8, 128, 10 ** 9) < 1 << 28
    assert f(64, 4, 8, 128, 10 ** 9, 10 ** 8, dtype=_lib.KH_F32) < 1 << 28


def _pool(bits=1, residual=True, shape=(2, 2, 16, 128)):
    return ops.empty_packed(shape, bits, residual, "cpu")


def test_python_layer_refuses_before_the_library():
    dk, dv, c = rademacher(128, 0), rademacher(128, 1), lloyd_max(1, 128)
    x, s = torch.zeros(3, 2, 128), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_append(x, x, _pool(), _pool(), s, dk, dv, c)
    q, t, n = torch.zeros(2, 4, 128), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_attention(q, _pool(), _pool(), t, n, dk, dv, c)
    with pytest.raises(ValueError, match="one shape"):
        ops._paged_pools(_pool(), _pool(shape=(2, 2, 8, 128)))
    with pytest.raises(ValueError, match="one shape"):
        ops._paged_pools(_pool(shape=(64, 128)), _pool(shape=(64, 128)))
    with pytest.raises(ValueError, match="residual"):
        ops._paged_pools(_pool(), _pool(residual=False))
    with pytest.raises(ValueError, match="bits=1"):
        ops._paged_pools(_pool(bits=2), _pool(bits=2))
