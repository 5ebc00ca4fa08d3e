"""Rotary positions, paged cache and the attention over it, as far as they go without a GPU: definitions, refusals, the C ABI's checks."""
import ctypes as C
import math
from fractions import Fraction

import pytest
import torch

import monarch_attention_b200 as ma
from monarch_attention_b200 import _cabi


@pytest.fixture(scope="module")
def lib():
    return _cabi.load()


@pytest.mark.parametrize("dim,base", [(64, 10000.0), (128, 500000.0), (2, 10000.0), (256, 1.0), (6, 1e-3)])
def test_turns_are_the_frequencies_in_fixed_point(dim, base):
    r = ma.RotaryPositions(dim, base=base)
    assert r.turns.dtype == torch.int64 and r.turns.shape == (dim // 2,) and r.magnitude == 1.0
    for i, (f, t) in enumerate(zip(r.frequencies, r.turns.tolist())):
        assert f == base ** (-2.0 * i / dim)
        # p * t / 2^64 turns is p * f radians, modulo one turn, to p * 2^-65 turns and what 64-bit floating point makes of pi
        for p in (1, 12345, 2 ** 30):
            got = (p * t) % 2 ** 64 / 2 ** 64
            want = math.fmod(float(Fraction(p) * Fraction(f) / (2 * Fraction(math.pi))), 1.0)
            off = abs(got - want)
            assert min(off, 1 - off) <= p * f * 2.0 ** -50 + p * 2.0 ** -64 + 2.0 ** -50 * (1 + p * f)


def test_scalings():
    plain = ma.RotaryPositions(64)
    linear = ma.RotaryPositions(64, scaling="linear", factor=4.0)
    assert all(a == b / 4.0 for a, b in zip(linear.frequencies, plain.frequencies))
    ntk = ma.RotaryPositions(64, scaling="ntk", factor=4.0)
    assert ntk.frequencies[0] == 1.0 and math.isclose(ntk.frequencies[-1], plain.frequencies[-1] / 4.0, rel_tol=1e-12)
    yarn = ma.RotaryPositions(64, scaling="yarn", factor=4.0, trained_length=4096)
    assert math.isclose(yarn.magnitude, 0.1 * math.log(4.0) + 1.0)
    for a, b in zip(yarn.frequencies, plain.frequencies):
        turns = 4096 * b / (2 * math.pi)
        assert a == b if turns >= 32 else math.isclose(a, b / 4.0) if turns <= 1 else b / 4.0 < a < b
    assert "yarn" in repr(yarn) and "64" in repr(plain)


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(dim=258), dict(dim=-2), dict(dim=64, pairs="other"), dict(dim=64, base=0.0), dict(dim=64, base=math.inf),
                                dict(dim=64, scaling="other"), dict(dim=64, scaling="linear", factor=0.0), dict(dim=2, scaling="ntk", factor=2.0),
                                dict(dim=64, scaling="yarn", factor=2.0), dict(dim=64, scaling="yarn", factor=2.0, trained_length=0)])
def test_rotary_definitions_are_checked(kw):
    with pytest.raises(ValueError):
        ma.RotaryPositions(**kw)


@pytest.mark.parametrize("kw", [dict(width=96), dict(page_size=8), dict(page_size=48), dict(pages=0), dict(heads=0)])
def test_cache_shapes_are_checked(kw):
    with pytest.raises(ValueError):
        ma.PagedKV.allocate(**{**dict(pages=2, heads=1, width=64, page_size=16, device="cpu"), **kw})


def test_allocated_cache():
    cache = ma.PagedKV.allocate(3, 2, 128, 32, device="cpu")
    assert cache.k.shape == cache.v.shape == (3, 2, 32, 128) and cache.k.dtype == torch.float8_e4m3fn
    assert cache.k_scale.shape == cache.v_scale.shape == (3, 2, 2) and cache.k_scale.dtype == torch.float32


def test_tensors_of_the_host_are_refused():
    r = ma.RotaryPositions(64)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    cache = ma.PagedKV.allocate(3, 2, 64, 16, device="cpu")
    table, lengths = torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ma.rotary_b200(q, None, r), lambda: ma.append_kv_b200(cache, q, q, table, lengths), lambda: ma.cached_attention_b200(q, cache, table, lengths),
                 lambda: ma.CachedAttention(r)(q, q, q, cache, table, lengths)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(TypeError):
        ma.rotary_b200(q, None, 64)
    with pytest.raises(TypeError):
        ma.append_kv_b200(cache, q, q, table, lengths, rotary=64)
    with pytest.raises(TypeError):
        ma.cached_attention_b200(q, (1, 2, 3, 4), table, lengths)
    with pytest.raises(ValueError):
        ma.CachedAttention(window=4, causal=False)
    with pytest.raises(ValueError):
        ma.CachedAttention(window=-1)


def rotary(dim=64, pairs=_cabi.PAIRS_HALF):
    turns = (C.c_uint64 * 128)()
    return _cabi.Rotary(dim, pairs, 1.0, turns)


def tensor(at=1 << 20, e=64, h=64, n=64):
    return _cabi.Tensor4(at, e, h, n)


def rotation(**kw):
    p = _cabi.Rotation(_cabi.ABI_VERSION, 1, 1, 0, 4, 64, _cabi.BF16, 0)
    p.q, p.q_out, p.rotary = tensor(), tensor(), rotary()
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw", [dict(abi_version=99), dict(E=0), dict(N=0), dict(D=0), dict(H=0), dict(H=-1), dict(dtype=9), dict(q=tensor(0)), dict(q=tensor((1 << 20) + 1)),
                                dict(q_out=tensor(n=-1)), dict(rotary=rotary(66)), dict(rotary=rotary(63)), dict(rotary=rotary(0)), dict(rotary=rotary(64, 5)),
                                dict(rotary=_cabi.Rotary(64, 0, 1.0, None)), dict(E=2 ** 16, N=2 ** 16)])
def test_rotation_problems_are_checked(lib, kw):
    assert lib.ma_b200_rotary_apply(C.byref(rotation(**kw)), None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_last_error()


def cache_struct(**kw):
    c = _cabi.Cache(1 << 20, 1 << 21, 1 << 22, 1 << 23, 8, 2, 32, 128, 8192, 4096, 128, 8192, 4096, 128, 4, 2, 4, 2)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def sequences(**kw):
    s = _cabi.Sequences(1 << 20, 4, 4, 1 << 20, None)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def attend(cache=None, seq=None, **kw):
    p = _cabi.Attend(_cabi.ABI_VERSION, 1, 4, 1, _cabi.BF16, 1, 0, 0.1, 0.0)
    p.q, p.out, p.cache, p.sequences = tensor(), tensor(), cache or cache_struct(), seq or sequences()
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=(1 << 20) + 8), dict(k_scale=(1 << 22) + 2), dict(pages=0), dict(page_size=8),
              dict(page_size=48), dict(k_stride_token=120), dict(v_stride_page=-16), dict(ks_stride_head=-1), dict(k_stride_page=2 ** 40)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_caches_are_checked(lib, kw):
    p = attend(cache_struct(**kw))
    assert lib.ma_b200_cache_attend(C.byref(p), 1 << 20, 1 << 40, None) == _cabi.INVALID_ARGUMENT
    a = _cabi.Append(_cabi.ABI_VERSION, 1, 0, 1, _cabi.BF16)
    a.k, a.v, a.cache, a.sequences = tensor(), tensor(), cache_struct(**kw), sequences()
    assert lib.ma_b200_cache_append(C.byref(a), None) == _cabi.INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(abi_version=99), dict(E=0), dict(N=0), dict(H=0), dict(H=3), dict(dtype=_cabi.F32), dict(seq=sequences(page_table=None)),
                                dict(seq=sequences(lengths=None)), dict(seq=sequences(table_pages=0)), dict(seq=sequences(table_stride=-1)), dict(N=1 << 30),
                                dict(E=1 << 30, H=64, N=64)])
def test_attention_problems_are_checked(lib, kw):
    p = attend(**kw)
    assert lib.ma_b200_cache_attend(C.byref(p), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_attend(None, 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT


def test_widths_and_rotations_that_the_cache_does_not_take(lib):
    assert lib.ma_b200_cache_attend(C.byref(attend(cache_struct(width=96))), 1 << 20, 1 << 60, None) == _cabi.UNSUPPORTED
    assert lib.ma_b200_cache_append(None, None) == _cabi.INVALID_ARGUMENT


def test_attention_scratch_is_host_arithmetic(lib):
    size = lambda **kw: lib.ma_b200_cache_attend_workspace_bytes(C.byref(attend(**kw)))  # noqa: E731
    assert size() == 256                                          # short sequences: nothing is split
    assert size(seq=sequences(table_pages=1000)) > 256            # long ones: pieces of heads
    assert size(seq=sequences(table_pages=1000), window=64) == 256   # a window makes them short
    assert size(N=200) == 256 and size(N=200, seq=sequences(table_pages=1000)) > 256
    assert size(H=3) == 0 and size(E=0) == 0


def test_status_of_a_device_that_had_no_call(lib):
    assert lib.ma_b200_poll_cache_status(0) == _cabi.OK and lib.ma_b200_poll_cache_status(-1) == _cabi.OK
    assert b"page" in lib.ma_b200_status_string(_cabi.DEVICE_BAD_SEQUENCE)


def test_positions_stay_below_2_to_the_31(lib):
    a = _cabi.Append(_cabi.ABI_VERSION, 1, 0, 1000, _cabi.BF16)
    a.k, a.v, a.cache, a.sequences = tensor(), tensor(), cache_struct(), sequences(table_pages=2 ** 26)
    assert lib.ma_b200_cache_append(C.byref(a), None) == _cabi.INVALID_ARGUMENT and b"2^31" in lib.ma_b200_last_error()


@pytest.mark.parametrize("softcap", [-1.0, 1e-30, 1e31, float("inf"), float("nan")])
def test_caps_that_leave_32_bits(lib, softcap):
    assert lib.ma_b200_cache_attend(C.byref(attend(softcap=softcap)), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
