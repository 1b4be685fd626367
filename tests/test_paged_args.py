"""fa_rotary and the fa_paged_* entry points reject bad arguments with the
documented status codes before touching the GPU (fake, never dereferenced
pointers), and the wrappers refuse what needs no GPU to see."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from flash_attn_volta import _capi

P, BAD = 0x10000, 0x10002


def _st(B, S, H, D):
    return (ctypes.c_int64 * 4)(S * H * D, H * D, D, 1)


@pytest.fixture(scope="module")
def lib():
    return _capi.load()


def _rotary(lib, **kw):
    a = dict(q=P, k=P, qo=P, ko=P, steps=P, factor=1.0, dim=64, flags=0, pos=P,
             ps=(ctypes.c_int64 * 2)(0, 1), B=2, S=4, H=4, Hk=2, D=128, qs=None, ks=None, qos=None,
             kos=None, dtype=0)
    a.update(kw)
    for n, h in (("qs", a["H"]), ("ks", a["Hk"]), ("qos", a["H"]), ("kos", a["Hk"])):
        a[n] = a[n] or _st(a["B"], a["S"], h, a["D"])
    return lib.fa_rotary(a["q"], a["k"], a["qo"], a["ko"], a["steps"], a["factor"], a["dim"],
                         a["flags"], a["pos"], a["ps"], a["B"], a["S"], a["H"], a["Hk"], a["D"],
                         a["qs"], a["ks"], a["qos"], a["kos"], a["dtype"], None)


@pytest.mark.parametrize("want,kw", [
    (_capi.FA_ERR_DTYPE, dict(dtype=2)), (_capi.FA_ERR_SHAPE, dict(B=0)),
    (_capi.FA_ERR_SHAPE, dict(H=0)), (_capi.FA_ERR_SHAPE, dict(Hk=-1)),
    (_capi.FA_ERR_HEAD_DIM, dict(D=60)), (_capi.FA_ERR_HEAD_DIM, dict(D=264)),
    (_capi.FA_ERR_HEAD_DIM, dict(dim=63)), (_capi.FA_ERR_HEAD_DIM, dict(dim=130)),
    (_capi.FA_ERR_HEAD_DIM, dict(dim=0)), (_capi.FA_ERR_NULL_POINTER, dict(steps=None)),
    (_capi.FA_ERR_NULL_POINTER, dict(pos=None)), (_capi.FA_ERR_NULL_POINTER, dict(q=None)),
    (_capi.FA_ERR_NULL_POINTER, dict(ko=None)), (_capi.FA_ERR_ALIGNMENT, dict(q=BAD)),
    (_capi.FA_ERR_ALIGNMENT, dict(pos=BAD)),
    (_capi.FA_ERR_ALIGNMENT, dict(pos=0x10004, flags=_capi.FA_ROTARY_POS64)),
    (_capi.FA_ERR_ALIGNMENT, dict(steps=0x10004)),
    (_capi.FA_ERR_SCALE, dict(factor=math.inf)),
    (_capi.FA_ERR_STRIDE, dict(ps=(ctypes.c_int64 * 2)(-4, 1))),
    (_capi.FA_ERR_STRIDE, dict(qs=(ctypes.c_int64 * 4)(2048, 512, 128, 2))),
    (_capi.FA_ERR_STRIDE, dict(ks=(ctypes.c_int64 * 4)(1024, 256, 130, 1))),
    (_capi.FA_ERR_STRIDE, dict(qos=(ctypes.c_int64 * 4)(0, 512, 128, 1))),
    (_capi.FA_ERR_STRIDE, dict(qos=(ctypes.c_int64 * 4)(2048, 512, 120, 1))),
    (_capi.FA_ERR_TOO_LARGE, dict(B=65536, S=65536, qs=_st(1, 1, 4, 128), ks=_st(1, 1, 2, 128))),
])
def test_rotary_statuses(lib, want, kw):
    assert _rotary(lib, **kw) == want


def _cache(**kw):
    a = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, pages=10, page_size=16, heads=2, width=4)
    a.update(kw)
    return _capi.PagedCacheStruct(*(a[n] for n, _ in _capi.PagedCacheStruct._fields_))


CACHE = [
    (_capi.FA_ERR_NULL_POINTER, dict(v_scales=None), {}), (_capi.FA_ERR_SHAPE, dict(pages=0), {}),
    (_capi.FA_ERR_SHAPE, dict(page_size=8), {}), (_capi.FA_ERR_SHAPE, dict(page_size=48), {}),
    (_capi.FA_ERR_SHAPE, dict(width=0), {}), (_capi.FA_ERR_SHAPE, dict(heads=0), {}),
    (_capi.FA_ERR_ALIGNMENT, dict(k_codes=0x10008), {}),
    (_capi.FA_ERR_ALIGNMENT, dict(v_scales=BAD), {}),
    (_capi.FA_ERR_TOO_LARGE, dict(width=1 << 30), {}),
    (_capi.FA_ERR_NULL_POINTER, {}, dict(table=None)), (_capi.FA_ERR_STRIDE, {}, dict(ts=-1)),
    (_capi.FA_ERR_SHAPE, {}, dict(B=0)), (_capi.FA_ERR_HEAD_DIM, {}, dict(D=96)),
    (_capi.FA_ERR_DTYPE, {}, dict(dtype=7)), (_capi.FA_ERR_TOO_LARGE, {}, dict(B=70000)),
]


def _append(lib, cache, **kw):
    a = dict(table=P, ts=4, k=P, v=P, q=P, qo=P, start=P, counts=None, steps=P, factor=1.0, dim=64,
             B=3, S=5, H=4, D=64, ks=None, qos=None, dtype=0)
    a.update(kw)
    kv = a["ks"] or _st(a["B"], a["S"], cache.heads, a["D"])
    qs = _st(a["B"], a["S"], a["H"], a["D"])
    return lib.fa_paged_append(cache, a["table"], a["ts"], a["k"], a["v"], a["q"], a["qo"],
                               a["start"], a["counts"], a["steps"], a["factor"], a["dim"], 0, a["B"],
                               a["S"], a["H"], a["D"], kv, kv, qs, a["qos"] or qs, a["dtype"], None)


@pytest.mark.parametrize("want,cache,kw", CACHE + [
    (_capi.FA_ERR_SHAPE, {}, dict(S=0)), (_capi.FA_ERR_SHAPE, {}, dict(H=0)),
    (_capi.FA_ERR_NULL_POINTER, {}, dict(k=None)), (_capi.FA_ERR_NULL_POINTER, {}, dict(start=None)),
    (_capi.FA_ERR_NULL_POINTER, {}, dict(qo=None)), (_capi.FA_ERR_HEAD_DIM, {}, dict(dim=66)),
    (_capi.FA_ERR_SCALE, {}, dict(factor=math.nan)), (_capi.FA_ERR_ALIGNMENT, {}, dict(counts=BAD)),
    (_capi.FA_ERR_STRIDE, {}, dict(ks=(ctypes.c_int64 * 4)(640, 128, 64, 2))),
    (_capi.FA_ERR_STRIDE, {}, dict(qos=(ctypes.c_int64 * 4)(1280, 256, 32, 1))),
])
def test_append_statuses(lib, want, cache, kw):
    assert _append(lib, _cache(**cache), **kw) == want


def _read(lib, cache, **kw):
    a = dict(table=P, ts=4, k=P, v=P, start=P, counts=None, B=3, n=5, D=64, dtype=0)
    a.update(kw)
    return lib.fa_paged_read(cache, a["table"], a["ts"], a["k"], a["v"], a["start"], a["counts"],
                             a["B"], a["n"], a["D"], a["dtype"], None)


@pytest.mark.parametrize("want,cache,kw", CACHE + [
    (_capi.FA_ERR_SHAPE, {}, dict(n=0)), (_capi.FA_ERR_NULL_POINTER, {}, dict(v=None)),
    (_capi.FA_ERR_ALIGNMENT, {}, dict(k=BAD)), (_capi.FA_ERR_NULL_POINTER, {}, dict(start=None)),
    (_capi.FA_ERR_TOO_LARGE, dict(heads=2048), dict(n=1 << 30, B=60000, width=1)),
])
def test_read_statuses(lib, want, cache, kw):
    kw = {n: v for n, v in kw.items() if n != "width"}
    assert _read(lib, _cache(**cache), **kw) == want


def _attn(lib, cache, **kw):
    a = dict(q=P, table=P, ts=4, lengths=P, counts=None, o=P, lse=None, ws=P, nb=1 << 40, B=3, Sq=2,
             H=4, D=64, qs=None, scale=0.1, dtype=0)
    a.update(kw)
    return lib.fa_paged_attn(a["q"], cache, a["table"], a["ts"], a["lengths"], a["counts"], a["o"],
                             a["lse"], a["ws"], a["nb"], a["B"], a["Sq"], a["H"], a["D"],
                             a["qs"] or _st(a["B"], a["Sq"], a["H"], a["D"]), a["scale"], a["dtype"],
                             None)


@pytest.mark.parametrize("want,cache,kw", CACHE + [
    (_capi.FA_ERR_SHAPE, {}, dict(Sq=0)), (_capi.FA_ERR_SHAPE, {}, dict(H=3)),
    (_capi.FA_ERR_NULL_POINTER, {}, dict(q=None)), (_capi.FA_ERR_NULL_POINTER, {}, dict(o=None)),
    (_capi.FA_ERR_NULL_POINTER, {}, dict(lengths=None)), (_capi.FA_ERR_ALIGNMENT, {}, dict(q=BAD)),
    (_capi.FA_ERR_ALIGNMENT, {}, dict(ws=BAD)), (_capi.FA_ERR_ALIGNMENT, {}, dict(lse=BAD)),
    (_capi.FA_ERR_WORKSPACE, {}, dict(ws=None)), (_capi.FA_ERR_WORKSPACE, {}, dict(nb=16)),
    (_capi.FA_ERR_SCALE, {}, dict(scale=math.inf)), (_capi.FA_ERR_TOO_LARGE, {}, dict(Sq=1 << 21)),
    (_capi.FA_ERR_STRIDE, {}, dict(qs=(ctypes.c_int64 * 4)(512, 256, 63, 1))),
])
def test_attend_statuses(lib, want, cache, kw):
    assert _attn(lib, _cache(**cache), **kw) == want


def test_workspace_sizes(lib):
    f = lib.fa_paged_attn_workspace_bytes
    assert f(1, 1, 8, 2, 64) > 0 and f(64, 4, 32, 8, 128) % 4 == 0
    for bad in ((0, 1, 8, 2, 64), (1, 0, 8, 2, 64), (1, 1, 7, 2, 64), (1, 1, 8, 2, 80), (1, 1, 8, 0, 64)):
        assert f(*bad) == 0


def test_frequencies_and_refusals():
    from flash_attn_volta import RotaryPositions
    from flash_attn_volta.forward import FlashAttnArgumentError
    make = lambda *a, **k: RotaryPositions(*a, device="cpu", **k)  # noqa: E731
    plain = make(64, base=500000.0).frequencies
    assert plain[0] == 1.0 and plain[16] == 500000.0 ** -0.5
    assert make(64, base=500000.0, scaling={"type": "linear", "factor": 4}).frequencies == \
        [f / 4 for f in plain]
    ntk = make(64, base=500000.0, scaling={"type": "ntk", "factor": 4}).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4)        # the slowest: 4 times slower
    y = make(64, base=10000.0, scaling={"type": "yarn", "factor": 4, "original_length": 4096})
    f = make(64).frequencies
    assert y.frequencies[0] == f[0] and math.isclose(y.frequencies[-1], f[-1] / 4)
    assert math.isclose(y.attention_factor, 0.1 * math.log(4) + 1)
    w = make(64, base=500000.0, scaling={"type": "wavelength", "factor": 8, "original_length": 8192,
                                         "low": 1, "high": 4}).frequencies
    for a, b in zip(plain, w):
        turns = 8192 * a / (2 * math.pi)
        assert math.isclose(b, a if turns > 4 else a / 8 if turns < 1 else b)
        assert a / 8 <= b * (1 + 1e-12) and b <= a * (1 + 1e-12)
    # a step is the frequency in turns, to 2^-64
    assert abs(make(2).steps.item() / 2 ** 64 - 1 / (2 * math.pi)) < 2 ** -53
    for bad in (lambda: make(63), lambda: make(0), lambda: make(258), lambda: make(64, base=0.0),
                lambda: make(64, base=math.nan), lambda: make(64, scaling={"type": "other"}),
                lambda: make(64, scaling={"type": "linear"}),
                lambda: make(64, scaling={"type": "linear", "factor": -2}),
                lambda: make(64, scaling={"type": "linear", "factor": 2, "low": 1}),
                lambda: make(64, scaling={"type": "yarn", "factor": 2}),
                lambda: make(64, scaling={"type": "factors", "factors": [1.0]}),
                lambda: make(64, scaling={"type": "wavelength", "factor": 2, "original_length": 10,
                                          "low": 4, "high": 1}),
                lambda: make(64, scaling="yarn")):
        with pytest.raises(FlashAttnArgumentError):
            bad()


def test_no_cpu_path():
    from flash_attn_volta import (PagedKVCache, RotaryPositions, append_paged,
                                  apply_rotary_positions, attend_paged, read_paged)
    from flash_attn_volta.forward import FlashAttnArgumentError
    cache = PagedKVCache(2, 16, 1, 32, torch.float16, device="cpu")
    k = torch.zeros((1, 1, 1, 32), dtype=torch.float16)
    t, n = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: append_paged(cache, k, k, t, n), lambda: attend_paged(k, cache, t, n),
                 lambda: read_paged(cache, t, n, 1),
                 lambda: apply_rotary_positions(k, None, n, RotaryPositions(32, device="cpu"))):
        with pytest.raises(FlashAttnArgumentError):
            call()


def test_handles_are_fixed_and_copy():
    """What the kernels are given sizes of cannot be exchanged under them; copies have
    tensors of their own."""
    import copy
    import pickle
    from flash_attn_volta import PagedKVCache, RotaryPositions
    cache = PagedKVCache(2, 16, 1, 32, torch.float16, device="cpu")
    rot = RotaryPositions(32, device="cpu")
    for obj, names in ((cache, ("k_codes", "head_dim", "num_pages", "dtype", "page_size")),
                       (rot, ("steps", "rotary_dim", "attention_factor", "interleaved"))):
        for n in names:
            with pytest.raises(AttributeError):
                setattr(obj, n, getattr(obj, n))
    cache._struct(3)
    other = copy.deepcopy(cache)
    assert other.k_codes.data_ptr() != cache.k_codes.data_ptr() and other.dtype == torch.float16
    assert other._struct(3)[0].k_codes == other.k_codes.data_ptr()
    again = pickle.loads(pickle.dumps(cache))
    assert again.num_pages == 2 and again.head_dim == 32 and torch.equal(again.v_codes, cache.v_codes)
    assert copy.copy(rot).steps is rot.steps and copy.deepcopy(rot).frequencies == rot.frequencies
    rot.frequencies.clear()
    assert len(rot.frequencies) == 16


def test_a_library_without_the_entry_points_is_named(tmp_path):
    """One of this version, built before they were added: rebuild it."""
    import subprocess
    src, out = tmp_path / "stub.c", tmp_path / "libfa_mi355x.so"
    src.write_text("int fa_abi_version(void) { return %d; }\n" % _capi.ABI_VERSION)
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(out)], check=True)
    with pytest.raises(_capi.LibraryNotBuilt, match="rebuild it"):
        _capi.load(str(out))


def test_numbers_out_of_range(lib):
    """Factors and frequencies that leave fp32's or Python's range are refused."""
    from flash_attn_volta import RotaryPositions
    from flash_attn_volta.forward import FlashAttnArgumentError
    assert _rotary(lib, factor=1e39) == _capi.FA_ERR_SCALE
    for kw in (dict(base=5e-324), dict(scaling={"type": "linear", "factor": 5e-324}),
               dict(base=1e300, scaling={"type": "ntk", "factor": 1e300}),
               dict(scaling={"type": "factors", "factors": [1.0] * 32, "attention_factor": 1e39})):
        with pytest.raises(FlashAttnArgumentError):
            RotaryPositions(64, device="cpu", **kw)
