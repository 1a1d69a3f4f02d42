"""The refusals of the beam-search entry points over the paged cache, which come
before any GPU work, and the plain forms that their GPU tests use.  CPU only."""
import ctypes

import numpy as np
import pytest

import beam_cases as B
from test_paged_cpu import ARG, UNSUPPORTED, A, _attn, _pages, _refused, needs_lib


def _filled(cls, **kw):
    f = {n: (A if t is ctypes.c_void_p else 1 << 30 if t is ctypes.c_size_t else 4) for n, t in cls._fields_}
    f.update(kw)
    return cls(**f)


def _select(**kw):
    import moehip as M
    return _filled(M.BeamSelect, **{**dict(n_groups=3, n_beam=4, vocab=100, ld=100), **kw})


def _fork(**kw):
    import moehip as M
    return _filled(M.PagedFork, **kw)


def _share(**kw):
    """as test_paged_cpu's _attn and _pages"""
    import moehip as M
    return _filled(M.PagedShare, **{**dict(T=3, n_req=5, max_pages=7, page_size=16, n_q=4, n_kv=2, head_dim=64, n_groups=2), **kw})


@needs_lib
@pytest.mark.parametrize("bad,want", [(dict(n_groups=-1), ARG), (dict(n_beam=0), ARG), (dict(vocab=0), ARG), (dict(ld=99), ARG), (dict(n_beam=65), UNSUPPORTED),
                                      (dict(n_groups=16384), UNSUPPORTED), (dict(vocab=(1 << 30) + 1, ld=1 << 31), UNSUPPORTED), (dict(work=A + 8), ARG),
                                      (dict(work_bytes=64), ARG)] + [({n: None}, ARG) for n in ("logits", "score", "parent", "token", "score_out", "done_out", "fresh", "work")],
                         ids=str)
def test_select_refused(bad, want):
    import moehip as M
    _refused(M.lib().moe_beam_select_dev(ctypes.byref(_select(**bad))), want)
    _refused(M.lib().moe_beam_select_dev(None), ARG)


@needs_lib
@pytest.mark.parametrize("bad,want", [(dict(n_req=-1), ARG), (dict(max_pages=0), ARG), (dict(n_pages=0), ARG), (dict(page_size=0), ARG), (dict(max_copies=-1), ARG),
                                      (dict(n_req=4097), UNSUPPORTED), (dict(max_copies=1 << 24), UNSUPPORTED), (dict(n_pages=1 << 28, page_size=8), ARG),
                                      (dict(max_pages=(1 << 29) + 1, page_size=2), ARG), (dict(work=A + 4), ARG), (dict(work_bytes=64), ARG)]
                         + [({n: None}, ARG) for n in ("parent", "held", "ring_at", "ring", "tables", "held_out", "ring_at_out", "tables_out", "copies", "status", "work")],
                         ids=str)
def test_fork_refused(bad, want):
    import moehip as M
    _refused(M.lib().moe_paged_fork_dev(ctypes.byref(_fork(**bad))), want)
    _refused(M.lib().moe_paged_fork_dev(None), ARG)


@needs_lib
def test_copy_refused():
    import moehip as M
    L = M.lib()
    two = lambda **kw: (M.Pages * 2)(_pages(), _pages(**kw))  # noqa: E731
    for args, want in (((A, -1, two(), 2), ARG), ((A, 1 << 24, two(), 2), ARG), ((A, 3, two(), -1), ARG), ((None, 3, two(), 2), ARG), ((A, 3, None, 2), ARG),
                       ((A, 3, two(k=None), 2), ARG), ((A, 3, two(head_dim=72), 2), UNSUPPORTED), ((A, 3, two(dtype=M.PAGE_F16), 2), UNSUPPORTED),
                       ((A, 3, two(n_pages=9), 2), UNSUPPORTED), ((A, 3, two(slot_stride=256), 2), UNSUPPORTED)):
        _refused(L.moe_paged_copy_dev(*args), want)
    assert L.moe_paged_copy_dev(None, 0, two(), 2) == 0 and L.moe_paged_copy_dev(A, 3, None, 0) == 0


SHARE = [(dict(T=-1), ARG), (dict(n_req=-1), ARG), (dict(max_pages=0), ARG), (dict(page_size=0), ARG), (dict(n_groups=-1), ARG), (dict(max_pages=(1 << 26) + 1), ARG),
         (dict(T=65537), UNSUPPORTED), (dict(n_groups=65537), UNSUPPORTED), (dict(n_q=5), ARG), (dict(n_kv=0), ARG), (dict(head_dim=40), ARG), (dict(head_dim=272), ARG),
         (dict(req=None, n_req=2), ARG), (dict(pos=None), ARG), (dict(tables=None), ARG), (dict(first=None), ARG), (dict(prefix=None), ARG), (dict(plan=None), ARG),
         (dict(plan=A + 8), ARG), (dict(plan_bytes=1), ARG)]


@needs_lib
@pytest.mark.parametrize("bad,want", SHARE, ids=str)
def test_share_refused(bad, want):
    import moehip as M
    L, s = M.lib(), _share(**bad)
    _refused(L.moe_paged_share_dev(ctypes.byref(s)), want)
    _refused(L.moe_paged_share_dev(None), ARG)
    _refused(L.moe_paged_attn_shared_dev(ctypes.byref(_attn()), ctypes.byref(_pages()), ctypes.byref(s)), want)


@needs_lib
@pytest.mark.parametrize("bad", [dict(T=2), dict(n_req=6), dict(max_pages=8), dict(page_size=8), dict(n_q=8), dict(n_kv=1), dict(head_dim=128), dict(req=2 * A), dict(pos=2 * A),
                                 dict(tables=2 * A)], ids=str)
def test_shared_attention_of_another_plan_refused(bad):
    import moehip as M
    _refused(M.lib().moe_paged_attn_shared_dev(ctypes.byref(_attn()), ctypes.byref(_pages()), ctypes.byref(_share(**bad))), ARG)


@needs_lib
@pytest.mark.parametrize("bad", [dict(T=-1), dict(n_q=0), dict(ldq=255), dict(ldo=255), dict(q=None), dict(out=None), dict(out=A), dict(work=None), dict(work=A + 8),
                                 dict(work_bytes=0)], ids=str)
def test_shared_attention_refused(bad):
    import moehip as M
    L, g, s = M.lib(), _pages(), _share()
    _refused(L.moe_paged_attn_shared_dev(ctypes.byref(_attn(**bad)), ctypes.byref(g), ctypes.byref(s)), ARG)
    _refused(L.moe_paged_attn_shared_dev(None, ctypes.byref(g), ctypes.byref(s)), ARG)
    _refused(L.moe_paged_attn_shared_dev(ctypes.byref(_attn()), None, ctypes.byref(s)), ARG)
    _refused(L.moe_paged_attn_shared_dev(ctypes.byref(_attn()), ctypes.byref(g), None), ARG)


@needs_lib
def test_shared_attention_of_too_many_blocks_refused():
    """2^24 rows' heads: more threads than a launch holds."""
    import moehip as M
    rows = dict(T=16384, n_req=16384, n_q=1024)
    a = _attn(**rows, ldq=1 << 16, ldo=1 << 16, work_bytes=1 << 60)
    g = _pages(n_kv=1024, head_stride=64, slot_stride=1 << 16, page_stride=1 << 20)
    s = _share(**rows, n_kv=1024, plan_bytes=1 << 60)
    _refused(M.lib().moe_paged_attn_shared_dev(ctypes.byref(a), ctypes.byref(g), ctypes.byref(s)), UNSUPPORTED)


@needs_lib
def test_work_of_refused_sizes():
    import moehip as M
    L = M.lib()
    assert L.moe_beam_select_work_bytes(1, 65, 100) == 0 and L.moe_beam_select_work_bytes(1, 4, 100) > 0
    assert L.moe_paged_fork_work_bytes(4097, 4, 4) == 0 and L.moe_paged_fork_work_bytes(4096, 4, 4) > 0
    assert L.moe_paged_share_plan_bytes(1 << 17, 1, 4, 2, 64) == 0 and L.moe_paged_attn_shared_work_bytes(4, 1, 5, 2, 64) == 0


def test_plain_fork_by_hand():
    """Two pages of four positions held by three requests: 0 and 1 share page 5; 2 ends; 1 becomes a copy of 0."""
    tables = np.array([[5, 1, -1], [5, 2, -1], [3, -1, -1]], np.int32)
    ring = np.array([9, 8, 7, 6, 4, 0, 0, 0, 0, 0], np.int32)
    got = B.fork([0, 0, -1], [6, 7, 3], tables, ring, [0, 5], 4, 3)
    assert got["status"] == B.OK
    assert got["tables"].tolist() == [[5, 1, -1], [5, 9, -1], [3, -1, -1]] and got["held"].tolist() == [6, 6, 0]
    assert got["copies"].tolist() == [[1, 9, 2], [-1, -1, -1], [-1, -1, -1]]
    assert got["ring_at"].tolist() == [1, 6] and got["ring"][5:7].tolist() == [3, 2]   # column by column


def test_plain_share_by_hand():
    tables = np.array([[4, 5, 6], [4, 5, 7], [4, 8, 7], [1, 2, 3]], np.int32)
    assert B.share([0, 1, 2, 3], [11, 9, 8, 5], tables, [0, 2, 3, 4], 4).tolist() == [8, 8, 4]
    assert B.share([0, 1, 2], [11, 3, 8], tables, [0, 3], 4).tolist() == [4]
    assert B.share([0, 1, -1, 2], [11, -1, 8, 11], tables, [0, 4], 4).tolist() == [4]
    assert B.share([0, 1], [11, 11], tables, [2, 0], 4).tolist() == [0]
