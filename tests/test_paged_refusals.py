"""Arguments that the paged-cache and sampling entry points refuse.  Every check runs on the
host before anything is launched, so these calls are made without a GPU; the pointers are
host memory that no refused call touches."""
import ctypes as C
import os

import numpy as np
import pytest

from rapidllm_amd import hip

RANGE, UNSUPPORTED = 6, 4
F32, F16, BF16, FP8 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(hip.LIB_PATH):
        pytest.skip("library not built (python -c 'import __graft_entry__ as g; g.build()')")
    return hip.lib()


BUF = np.zeros(4096, np.uint8)
P = (BUF.ctypes.data + 255) // 256 * 256


def cache(**kw):
    d = dict(k=P, v=P, layer_stride=4 * 2 * 16 * 128, n_layers=1, n_pages=4, page_size=16, n_kv=2, head_dim=128,
             dtype=F16)
    d.update(kw)
    return hip.RlPagedCache(*(d[f] for f, _ in hip.RlPagedCache._fields_))


def append(L, c, **kw):
    a = dict(layer=0, dtype=F16, q=P, q_row=1024, q_head=128, k=P, k_row=1024, k_head=128, v=P, v_row=1024, v_head=128,
             qn=P, kn=P, norm=1, eps=1e-6, rot=64, theta=1e6, pos=P, slots=P, rows=3, nq=4, out=P)
    a.update(kw)
    return L.rl_hip_paged_append(c, *a.values(), None)


def attn(L, c, **kw):
    a = dict(layer=0, dtype=F16, q=P, q_row=512, q_head=128, gate=None, g_row=0, g_head=0, table=P, width=4, ctx=P,
             start=P, n_seq=2, rows=3, max_rows=2, mask=None, words=0, nq=4, scale=0.1, out=P, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return L.rl_hip_tree_attn(c, *a.values(), None)


def accept(L, c, **kw):
    a = dict(table=P, width=4, ctx=P, start=P, n_seq=2, rows=3, parents=P, toks=P, samples=P, path=P, cap=4, n=P,
             nxt=P, ctx_out=P + 64)
    a.update(kw)
    return L.rl_hip_tree_accept(c, *a.values(), None)


def sample(L, **kw):
    a = dict(dtype=F32, logits=P, ld=100, rows=2, V=100, t=None, k=None, p=None, mp=None, u=P, idx=P, prob=None, ws=P,
             ws_bytes=1 << 40)
    a.update(kw)
    return L.rl_hip_sample_rows(*a.values(), None)


BAD_CACHES = [(dict(k=None), RANGE), (dict(v=None), RANGE), (dict(head_dim=96), UNSUPPORTED),
              (dict(dtype=F32), UNSUPPORTED), (dict(dtype=FP8), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
              (dict(page_size=0), UNSUPPORTED), (dict(page_size=8192), UNSUPPORTED), (dict(n_pages=0), RANGE),
              (dict(n_kv=0), RANGE), (dict(n_layers=2, layer_stride=8), RANGE), (dict(layer_stride=12), RANGE),
              (dict(k=P + 2), RANGE)]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_descriptions(L, bad, code):
    c = cache(**bad)
    assert append(L, c) == code
    assert attn(L, c) == code
    assert accept(L, c) == code
    assert b"append" in (append(L, c), L.rl_hip_last_error())[1]


@pytest.mark.parametrize("bad,code", [
    (dict(layer=1), RANGE), (dict(layer=-1), RANGE), (dict(dtype=BF16), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED),
    (dict(q=None), RANGE), (dict(out=None), RANGE), (dict(k=None), RANGE), (dict(v=None), RANGE),
    (dict(pos=None), RANGE), (dict(slots=None), RANGE), (dict(q=P + 4), RANGE), (dict(k_row=1022), RANGE),
    (dict(v_head=130), RANGE), (dict(rot=4), RANGE), (dict(rot=136), RANGE), (dict(rot=-8), RANGE),
    (dict(theta=0.0), RANGE), (dict(theta=float("nan")), RANGE), (dict(eps=-1.0), RANGE),
    (dict(eps=float("nan")), RANGE), (dict(rows=-1), RANGE), (dict(nq=-1), RANGE), (dict(out=P + 2), RANGE)])
def test_append_refuses(L, bad, code):
    assert append(L, cache(), **bad) == code


def test_rows_of_another_type_than_the_cache(L):
    assert append(L, cache(dtype=BF16), dtype=F32) == UNSUPPORTED
    assert append(L, cache(dtype=BF16), dtype=F16) == UNSUPPORTED
    assert attn(L, cache(dtype=BF16), dtype=F32) == UNSUPPORTED
    assert attn(L, cache(), dtype=BF16) == UNSUPPORTED


@pytest.mark.parametrize("bad,code", [
    (dict(layer=1), RANGE), (dict(q=None), RANGE), (dict(table=None), RANGE), (dict(ctx=None), RANGE),
    (dict(start=None), RANGE), (dict(out=None), RANGE), (dict(ws=None), RANGE), (dict(ws_bytes=8), RANGE),
    (dict(nq=3), RANGE), (dict(nq=0), RANGE), (dict(nq=130), RANGE), (dict(width=0), RANGE),
    (dict(width=1 << 30), RANGE), (dict(mask=P, words=0), RANGE), (dict(scale=float("nan")), RANGE),
    (dict(scale=float("inf")), RANGE), (dict(q=P + 4), RANGE), (dict(q_head=130), RANGE),
    (dict(gate=P + 2, g_row=512, g_head=128), RANGE), (dict(out=P + 8), RANGE), (dict(rows=-1), RANGE),
    (dict(n_seq=-1), RANGE), (dict(max_rows=-1), RANGE)])
def test_attn_refuses(L, bad, code):
    assert attn(L, cache(), **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(table=None), RANGE), (dict(ctx=None), RANGE), (dict(start=None), RANGE), (dict(parents=None), RANGE),
    (dict(toks=None), RANGE), (dict(samples=None), RANGE), (dict(path=None), RANGE), (dict(n=None), RANGE),
    (dict(nxt=None), RANGE), (dict(ctx_out=None), RANGE), (dict(ctx_out=P), RANGE), (dict(cap=0), RANGE),
    (dict(cap=4097), RANGE), (dict(width=0), RANGE), (dict(width=1 << 30), RANGE), (dict(n_seq=-1), RANGE),
    (dict(rows=-1), RANGE)])
def test_accept_refuses(L, bad, code):
    assert accept(L, cache(), **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=FP8), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(logits=None), RANGE), (dict(u=None), RANGE),
    (dict(idx=None), RANGE), (dict(ws=None), RANGE), (dict(ws_bytes=8), RANGE), (dict(ld=99), RANGE),
    (dict(V=0), RANGE), (dict(V=(1 << 24) + 1, ld=1 << 25), RANGE), (dict(rows=-1), RANGE),
    (dict(logits=P + 2), RANGE), (dict(ws=P + 8), RANGE)])
def test_sample_refuses(L, bad, code):
    assert sample(L, **bad) == code


def test_empty_calls_do_nothing(L):
    """No rows or no sequences: accepted, nothing launched, nothing read."""
    assert append(L, cache(), rows=0, q=None, k=None, v=None, pos=None, slots=None, out=None) == 0
    assert attn(L, cache(), rows=0, q=None, out=None, ws=None) == 0
    assert attn(L, cache(), n_seq=0) == 0
    assert accept(L, cache(), n_seq=0, path=None) == 0
    assert sample(L, rows=0, logits=None, u=None) == 0


def test_workspace_sizes(L):
    """Positive, and not smaller for more rows or sequences."""
    a = [L.rl_hip_tree_attn_workspace_bytes(24, 4, 256, b, r) for b, r in ((1, 1), (8, 1), (8, 64), (64, 64))]
    assert a[0] > 0 and a == sorted(a)
    s = [L.rl_hip_sample_workspace_bytes(r, v) for r, v in ((1, 1000), (1, 248320), (128, 248320))]
    assert s[0] > 0 and s == sorted(s)


def test_attn_mask_alignment_and_size_limits(L):
    assert attn(L, cache(), mask=P + 4, words=1) == RANGE
    # more rows than 32-bit row numbers hold, more units of work than 32 bits count
    big = cache(n_pages=1 << 20, page_size=4096, layer_stride=0)
    assert attn(L, big) == UNSUPPORTED
    assert attn(L, cache(), width=1 << 26, n_seq=4000) == UNSUPPORTED


@pytest.mark.parametrize("nq,nkv,hd", [(24, 4, 256), (32, 8, 128), (64, 1, 64)])
def test_attn_workspace_serves_fewer_rows(L, nq, nkv, hd):
    """Non-decreasing over max_rows, so that one workspace serves every smaller step."""
    a = [L.rl_hip_tree_attn_workspace_bytes(nq, nkv, hd, 8, r) for r in range(1, 700)]
    assert a == sorted(a)


def test_tables_of_more_than_2_30_positions(L):
    assert attn(L, cache(), width=(1 << 26) + 1) == RANGE
    assert accept(L, cache(), width=(1 << 26) + 1) == RANGE
