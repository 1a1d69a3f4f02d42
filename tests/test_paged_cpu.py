"""The paged cache's index arithmetic (csrc/paged.h, compiled for the host) and
the refusals of its entry points, which come before any GPU work.  CPU only."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "moe.cc_amd", "libmoehip.so")
ARG, UNSUPPORTED = 2, 4

needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="libmoehip.so not built")


def test_index_arithmetic(tmp_path):
    exe = str(tmp_path / "paged_index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    os.path.join(ROOT, "tests", "paged_index.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr


A = 1 << 20   # any 16-byte aligned address: a refused call touches none


def _pages(**kw):
    import moehip as M
    f = dict(k=A, v=A, dtype=M.PAGE_BF16, n_pages=10, page_size=16, n_kv=2, head_dim=64, page_stride=2048, head_stride=64,
             slot_stride=128, k_scale=None, v_scale=None)
    f.update(kw)
    return M.Pages(**f)


def _plan(**kw):
    import moehip as M
    f = {n: (A if t is ctypes.c_void_p else 4) for n, t in M.PagedPlan._fields_}
    f.update(kw)
    return M.PagedPlan(**f)


def _heads(**kw):
    import moehip as M
    f = dict(qkv=A, ld=1024, T=3, n_q=4, pos=A, slot=A, q_norm=A, k_norm=A, eps=1e-6, rope_cos=A, rope_sin=A, rope_len=100,
             rope_dim=64, q_out=2 * A, ldq=256)
    f.update(kw)
    return M.PagedHeads(**f)


def _attn(**kw):
    import moehip as M
    f = dict(q=A, ldq=256, T=3, n_q=4, req=A, pos=A, tables=A, n_req=5, max_pages=7, scale=0.125, out=2 * A, ldo=256, work=3 * A,
             work_bytes=1 << 30)
    f.update(kw)
    return M.PagedAttn(**f)


PAGES = [(dict(k=None), ARG), (dict(v=None), ARG), (dict(dtype=2), ARG), (dict(dtype=-1), ARG), (dict(n_pages=0), ARG), (dict(page_size=0), ARG),
         (dict(n_kv=0), ARG), (dict(n_pages=1 << 20, page_size=1 << 11), ARG), (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=72), UNSUPPORTED),
         (dict(head_dim=272), UNSUPPORTED), (dict(slot_stride=63), ARG), (dict(slot_stride=132), ARG), (dict(head_stride=-64), ARG),
         (dict(page_stride=0), ARG), (dict(n_pages=1 << 20, page_stride=1 << 30), ARG), (dict(k=A + 8), ARG), (dict(v=A + 4), ARG), (dict(k_scale=A), ARG), (dict(v_scale=A), ARG)]


def _refused(st, want):
    import moehip as M
    assert st == want and M.lib().moe_last_error()


@needs_lib
@pytest.mark.parametrize("bad,want", PAGES, ids=lambda v: str(v))
def test_pages_refused(bad, want):
    import moehip as M
    L = M.lib()
    g = _pages(**bad)
    _refused(L.moe_paged_heads_dev(ctypes.byref(_heads()), ctypes.byref(g)), want)
    _refused(L.moe_paged_attn_dev(ctypes.byref(_attn()), ctypes.byref(g)), want)


@needs_lib
@pytest.mark.parametrize("bad", [dict(n_req=-1), dict(max_pages=0), dict(n_pages=0), dict(page_size=0), dict(max_tokens=-1),
                                 dict(n_req=1 << 24), dict(max_tokens=1 << 24), dict(n_pages=1 << 28, page_size=8), dict(max_pages=(1 << 29) + 1, page_size=2)]
                         + [{n: None} for n in ("fresh", "held", "ring_at", "ring", "tables", "held_out", "ring_at_out", "starts", "req", "pos",
                                                "slot", "status")], ids=str)
def test_plan_refused(bad):
    import moehip as M
    _refused(M.lib().moe_paged_plan_dev(ctypes.byref(_plan(**bad))), ARG)
    _refused(M.lib().moe_paged_plan_dev(None), ARG)


@needs_lib
@pytest.mark.parametrize("bad", [dict(T=-1), dict(n_q=0), dict(n_q=3), dict(ld=511), dict(ldq=255), dict(rope_dim=3), dict(rope_dim=66),
                                 dict(rope_dim=-2), dict(rope_len=-1), dict(qkv=None), dict(pos=None), dict(slot=None), dict(q_out=None),
                                 dict(rope_cos=None), dict(rope_sin=None), dict(q_out=A), dict(T=1 << 30)], ids=str)
def test_heads_refused(bad):
    import moehip as M
    L, g = M.lib(), _pages()
    _refused(L.moe_paged_heads_dev(ctypes.byref(_heads(**bad)), ctypes.byref(g)), ARG)
    _refused(L.moe_paged_heads_dev(None, ctypes.byref(g)), ARG)
    _refused(L.moe_paged_heads_dev(ctypes.byref(_heads()), None), ARG)


@needs_lib
@pytest.mark.parametrize("bad", [dict(T=-1), dict(n_q=0), dict(n_q=5), dict(ldq=255), dict(ldo=255), dict(n_req=-1), dict(max_pages=0),
                                 dict(max_pages=(1 << 26) + 1), dict(req=None, n_req=2), dict(q=None), dict(pos=None), dict(tables=None),
                                 dict(T=1 << 24, n_req=1 << 25), dict(out=None), dict(out=A), dict(work=None), dict(work=A + 8), dict(work_bytes=0)], ids=str)
def test_attn_refused(bad):
    import moehip as M
    L, g = M.lib(), _pages()
    _refused(L.moe_paged_attn_dev(ctypes.byref(_attn(**bad)), ctypes.byref(g)), ARG)
    _refused(L.moe_paged_attn_dev(None, ctypes.byref(g)), ARG)
    _refused(L.moe_paged_attn_dev(ctypes.byref(_attn()), None), ARG)


@needs_lib
def test_empty_calls():
    """No rows: done without touching the GPU."""
    import moehip as M
    L, g = M.lib(), _pages()
    assert L.moe_paged_heads_dev(ctypes.byref(_heads(T=0, qkv=None)), ctypes.byref(g)) == 0
    assert L.moe_paged_attn_dev(ctypes.byref(_attn(T=0, q=None, work=None)), ctypes.byref(g)) == 0
