"""Drafted trees, their acceptance and forked sequences, as far as they go without a GPU: definitions, refusals, the C ABI's checks."""
import ctypes as C

import pytest
import torch

import monarch_attention_b200 as ma
from drafts_reference import accepted, forked, line, power_for
from monarch_attention_b200 import _cabi
from test_decoder_host import BAD_CACHES, attend, cache_struct, sequences, tensor


@pytest.fixture(scope="module")
def lib():
    return _cabi.load()


def tree(parents=1 << 20, stride=8):
    return _cabi.Tree(parents, stride)


def caches(n=1, **kw):
    return (_cabi.Cache * n)(*(cache_struct(**kw) for _ in range(n)))


def accept(c=None, seq=None, t=None, **kw):
    c = c or caches()
    p = _cabi.Accept(_cabi.ABI_VERSION, 1, 8, len(c), c, seq or sequences(), t or tree())
    p.drafted, p.answers, p.drafted_stride, p.answers_stride, p.ids_i64 = 1 << 20, 1 << 20, 8, 8, 1
    p.new_lengths, p.path, p.answer = 1 << 20, 1 << 20, 1 << 20
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def fork(c=None, **kw):
    c = c or caches()
    p = _cabi.Fork(_cabi.ABI_VERSION, 2, len(c), c, 1 << 20, 1 << 20, 4, 4, 1 << 20, None, None, 1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def append(**kw):
    a = _cabi.Append(_cabi.ABI_VERSION, 1, 0, 4, _cabi.BF16)
    a.k, a.v, a.cache, a.sequences = tensor(), tensor(), cache_struct(), sequences()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("t,N,code", [(None, 4, _cabi.INVALID_ARGUMENT), (tree(parents=None), 4, _cabi.INVALID_ARGUMENT), (tree(stride=-1), 4, _cabi.INVALID_ARGUMENT), (tree(), 513, _cabi.UNSUPPORTED)])
def test_trees_are_checked(lib, t, N, code):
    ref = C.byref(t) if t is not None else None
    assert lib.ma_b200_cache_attend_tree(C.byref(attend(N=N)), ref, 1 << 20, 1 << 60, None) == code
    assert lib.ma_b200_cache_append_tree(C.byref(append(N=N)), ref, None) == code
    assert lib.ma_b200_last_error()
    if t is not None:
        assert lib.ma_b200_cache_accept(C.byref(accept(t=t, N=N)), None) == code


def test_trees_keep_the_checks_of_the_calls_without(lib):
    assert lib.ma_b200_cache_attend_tree(None, C.byref(tree()), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_append_tree(None, C.byref(tree()), None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_attend_tree(C.byref(attend(causal=0)), C.byref(tree()), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_attend_tree(C.byref(attend(H=3)), C.byref(tree()), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_append_tree(C.byref(append(dtype=_cabi.F32)), C.byref(tree()), None) == _cabi.INVALID_ARGUMENT


def test_scratch_of_trees_is_host_arithmetic(lib):
    size = lambda **kw: lib.ma_b200_cache_attend_tree_workspace_bytes(C.byref(attend(**kw)))  # noqa: E731
    assert size() == size(N=8) == 256 and size(N=200) == 256                       # short sequences: nothing is split
    few, many = size(N=8, seq=sequences(table_pages=1000)), size(N=200, seq=sequences(table_pages=1000))
    assert few == lib.ma_b200_cache_attend_workspace_bytes(C.byref(attend(N=8, seq=sequences(table_pages=1000)))) > 256
    assert many >= 148 * 256 * (128 + 2) * 4                                       # a piece for each SM
    assert size(H=3) == 0 and size(E=0) == 0
    p = attend(N=200, seq=sequences(table_pages=1000))
    assert lib.ma_b200_cache_attend_tree(C.byref(p), C.byref(tree()), 1 << 20, many - 1, None) in (_cabi.WORKSPACE_TOO_SMALL, _cabi.CUDA_ERROR)   # (no device here)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_caches_are_checked(lib, kw):
    for c in (caches(**kw), (_cabi.Cache * 2)(cache_struct(), cache_struct(**kw))):
        assert lib.ma_b200_cache_accept(C.byref(accept(c)), None) == _cabi.INVALID_ARGUMENT
        assert lib.ma_b200_cache_fork(C.byref(fork(c)), 1 << 20, 1 << 40, None) == _cabi.INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(pages=9), dict(heads=3), dict(page_size=64), dict(width=64), dict(k_stride_token=256), dict(v_stride_page=16384), dict(ks_stride_page=8), dict(vs_stride_head=4)])
def test_layers_that_differ_are_refused(lib, kw):
    c = (_cabi.Cache * 3)(cache_struct(), cache_struct(), cache_struct(**kw))
    assert lib.ma_b200_cache_accept(C.byref(accept(c)), None) == _cabi.INVALID_ARGUMENT and b"layers" in lib.ma_b200_last_error()
    assert lib.ma_b200_cache_fork(C.byref(fork(c)), 1 << 20, 1 << 40, None) == _cabi.INVALID_ARGUMENT and b"layers" in lib.ma_b200_last_error()


@pytest.mark.parametrize("kw", [dict(abi_version=99), dict(E=0), dict(N=0), dict(layers=0), dict(caches=None), dict(drafted=None), dict(answers=None), dict(new_lengths=None), dict(path=None),
                                dict(answer=None), dict(drafted=(1 << 20) + 4), dict(drafted_stride=-1), dict(seq=sequences(lengths=None)), dict(seq=sequences(page_table=None)),
                                dict(N=512, seq=sequences(table_pages=1 << 27))])
def test_acceptance_is_checked(lib, kw):
    assert lib.ma_b200_cache_accept(C.byref(accept(**kw)), None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_accept(None, None) == _cabi.INVALID_ARGUMENT


@pytest.mark.parametrize("kw", [dict(abi_version=99), dict(E=0), dict(layers=0), dict(caches=None), dict(table_pages=0), dict(page_uses=None), dict(page_table=None), dict(lengths=None), dict(room_all=-1),
                                dict(table_stride=3), dict(table_stride=-1), dict(E=1 << 20, table_pages=1 << 12, table_stride=1 << 12)])
def test_forks_are_checked(lib, kw):
    assert lib.ma_b200_cache_fork(C.byref(fork(**kw)), 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_fork(None, 1 << 20, 1 << 60, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_fork_workspace_bytes(None) == 0


def test_fork_scratch(lib):
    need = lib.ma_b200_cache_fork_workspace_bytes(C.byref(fork()))
    assert 0 < need < 4096
    assert lib.ma_b200_cache_fork_workspace_bytes(C.byref(fork(E=100, table_pages=1000))) >= 4 * 100 * 1000
    assert lib.ma_b200_cache_fork(C.byref(fork()), 1 << 20, need - 1, None) == _cabi.WORKSPACE_TOO_SMALL
    assert lib.ma_b200_cache_fork(C.byref(fork()), (1 << 20) + 16, need, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_fork(C.byref(fork()), None, need, None) == _cabi.INVALID_ARGUMENT
    assert lib.ma_b200_cache_fork_workspace_bytes(C.byref(fork(E=0))) == 0


def test_tensors_of_the_host_are_refused():
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    cache = ma.PagedKV.allocate(3, 2, 64, 16, device="cpu")
    table, lengths, parents = torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([[-1, 0, 1]], dtype=torch.int32)
    for call in (lambda: ma.append_kv_b200(cache, q, q, table, lengths, parents=parents), lambda: ma.cached_attention_b200(q, cache, table, lengths, parents=parents),
                 lambda: ma.CachedAttention()(q, q, q, cache, table, lengths, None, parents), lambda: ma.accept_drafts_b200(cache, table, lengths, None, parents, parents, parents),
                 lambda: ma.fork_sequences_b200([cache], torch.zeros(3, dtype=torch.int32), table, lengths)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(TypeError):
        ma.cached_attention_b200(q, cache, table, lengths, parents=[[-1, 0, 1]])
    with pytest.raises(TypeError):
        ma.accept_drafts_b200([cache.k], table, lengths, None, parents, parents, parents)
    with pytest.raises(TypeError):
        ma.fork_sequences_b200(5, lengths, table, lengths)
    with pytest.raises(ValueError):
        ma.fork_sequences_b200([], lengths, table, lengths)


def test_definitions():
    assert line([-1, 0, 0, 2, 9], 3) == [3, 2, 0] and line([-1, 0, 0, 2, 9], 4) == [4]
    assert accepted([-1, 0, 0, 2, 2], [5, 6, 7, 8, 8], [7, 0, 8, 1, 1], 5) == [0, 2, 3] and accepted([-1], [5], [5], 0) == []
    assert power_for(448.0) == 1.0 and power_for(448.1) == 2.0 and power_for(0.0) == 2.0 ** -40
    # two rows of 20 tokens on pages of 16: row 1 goes on from row 0, whose first page they share; its own two are free again, the lowest is taken
    uses, table, lengths, copies = forked([1, 1, 1, 1, 0], [[3, 1, -1], [0, 2, -1]], [20, 20], [0, 0], [0, 0], 16)
    assert (uses, table, lengths, copies) == ([1, 1, 0, 2, 0], [[3, 1, -1], [3, 0, -1]], [20, 20], [(1, 0, 4)])
    # exchanged; ended with room for another
    assert forked([1, 1], [[0], [1]], [5, 6], [1, 0], [0, 0], 16)[:3] == ([1, 1], [[1], [0]], [6, 5])
    assert forked([1, 1, 0], [[0, -1], [1, -1]], [5, 6], [0, -1], [0, 17], 16)[:3] == ([1, 1, 1], [[0, -1], [1, 2]], [5, 0])
