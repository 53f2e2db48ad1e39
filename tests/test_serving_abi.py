"""CPU: argument checks of the serving entry points (norm and rotation, rotated paged
append, shared-prefix decode attention) before anything touches the GPU, the workspace
query, and the Python front ends' refusal of CPU tensors."""
import ctypes

import pytest
import torch

from bitcache_b200 import _lib, planes

OK, HEAD_DIM, ARG, ALIGN, WORKSPACE, UNSUPPORTED, TOO_LARGE = range(7)
P = 1 << 20  # a well-aligned address that nothing reads


def heads(at=P, dim=128, n=4):
    return _lib.Heads(at, n * dim, dim)


def rope(**kw):
    a = dict(cos=P, sin=P, q_weight=None, k_weight=None, n_positions=64, rotary_dim=128, interleaved=0, eps=1e-6) | kw
    return _lib.Rope(*(a[name] for name, _ in _lib.Rope._fields_))


def kv(at=P):
    return _lib.KVPlanes(at, at, at, at)


def table(page_size=128, n_pages=4, max_pages=2, pages=P):
    return _lib.PageTable(pages, max_pages, page_size, n_pages)


def norm_rope(**kw):
    a = dict(q=heads(), k=heads(), pos=P, rope=rope(), qo=P, ko=P, n=2, hq=4, hkv=4, d=128, t=0, to=0) | kw
    return _lib.load().bc_qk_norm_rope(*a.values(), None)


def append(**kw):
    a = dict(q=heads(), k=heads(), v=heads(), ids=P, pos=P, rope=rope(), qo=P, K=kv(), V=kv(), pt=table(), kh=None,
             vh=None, n=2, seqs=1, hq=4, hkv=4, d=128, t=0, mode=planes.RES_FP32_SCALE) | kw
    return _lib.load().bc_append_qkv_paged(*a.values(), None)


def attend(**kw):
    a = dict(q=P, K=kv(), V=kv(), pt=table(), lens=P, pre=P, out=P, seqs=8, groups=2, hkv=2, group=4, d=128,
             mode=planes.MODE_COMPENSATED, ws=P, bytes=1 << 40) | kw
    return _lib.load().bc_decode_attention_shared(*a.values(), None)


@pytest.mark.parametrize("call", [norm_rope, append, attend])
@pytest.mark.parametrize("d", [0, 16, 33, 288, -32])
def test_head_dim(call, d):
    assert call(d=d) == HEAD_DIM


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(hq=-1), dict(hkv=-1), dict(t=3), dict(to=-1), dict(pos=None), dict(qo=None), dict(ko=None),
    dict(q=heads(None)), dict(k=heads(None)), dict(rope=rope(cos=None)), dict(rope=rope(sin=None)),
    dict(rope=rope(rotary_dim=3)), dict(rope=rope(rotary_dim=130)), dict(rope=rope(n_positions=-1))])
def test_norm_rope_arguments(bad):
    assert norm_rope(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(q=heads(P + 1)), dict(pos=P + 2), dict(qo=P + 1), dict(ko=P + 2, to=2)])
def test_norm_rope_alignment(bad):
    assert norm_rope(**bad) == ALIGN


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(seqs=-1), dict(hq=-1), dict(hkv=0), dict(t=7), dict(mode=5), dict(ids=None), dict(pos=None),
    dict(qo=None), dict(kh=P), dict(vh=P), dict(K=kv(None)), dict(V=kv(None)), dict(v=heads(None)),
    dict(pt=table(pages=None)), dict(pt=table(page_size=64)), dict(pt=table(n_pages=0)), dict(pt=table(max_pages=0))])
def test_append_arguments(bad):
    assert append(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(K=kv(P + 8)), dict(V=kv(P + 4)), dict(ids=P + 2), dict(qo=P + 1), dict(kh=P + 1, vh=P)])
def test_append_alignment(bad):
    assert append(**bad) == ALIGN


@pytest.mark.parametrize("bad", [
    dict(seqs=-1), dict(groups=0), dict(groups=3), dict(hkv=0), dict(group=0), dict(mode=4), dict(q=None),
    dict(lens=None), dict(out=None), dict(K=kv(None)), dict(V=kv(None)), dict(pt=table(pages=None)),
    dict(pt=table(page_size=100)), dict(pt=table(n_pages=0)), dict(pt=table(max_pages=-1))])
def test_attention_arguments(bad):
    assert attend(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(q=P + 1), dict(K=kv(P + 8)), dict(lens=P + 1), dict(pre=P + 2), dict(ws=P + 8)])
def test_attention_alignment(bad):
    assert attend(**bad) == ALIGN


def test_attention_sizes():
    assert attend(d=96) == UNSUPPORTED
    assert attend(seqs=1 << 20, groups=1, hkv=1 << 10, group=1 << 5) == TOO_LARGE
    assert attend(ws=None) == WORKSPACE
    need = _lib.load().bc_decode_shared_workspace_bytes(8, 2, 2, 4, 128)
    assert attend(bytes=need - 1) == WORKSPACE


def test_empty_calls_do_nothing():
    none = dict(q=heads(None), k=heads(None), pos=None)
    assert norm_rope(n=0, qo=None, ko=None, **none) == OK
    assert norm_rope(hq=0, hkv=0) == OK
    assert append(n=0, v=heads(None), ids=None, qo=None, **none) == OK
    assert attend(seqs=0, groups=0, q=None, lens=None, out=None) == OK


def test_workspace_query():
    query = _lib.load().bc_decode_shared_workspace_bytes
    for bad in ((0, 1, 8, 4, 128), (8, 3, 8, 4, 128), (8, 0, 8, 4, 128), (8, 1, 0, 4, 128), (8, 1, 8, 0, 128), (8, 1, 8, 4, 96)):
        assert query(*bad) == 0
    for d in (32, 64, 128, 256):
        for seqs, groups in ((1, 1), (16, 1), (16, 4), (128, 16)):
            n = query(seqs, groups, 8, 4, d)
            # at least one record (a float per dim, and two) of every query row's own keys and of its prefix
            assert n >= 2 * seqs * 8 * 4 * (d + 4) * 4


def test_python_front_ends_refuse_cpu_tensors():
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(2, 2, 64, dtype=torch.float16)
    pos, none = torch.zeros(2, dtype=torch.int32), planes.Rope(None, None)
    pool = planes.Planes.empty(4, 128, 64, True, torch.device("cpu"))
    pt = planes.PageTable(torch.zeros(4, 2, dtype=torch.int32), 128, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        planes.qk_norm_rope(q, k, pos, none)
    with pytest.raises(RuntimeError, match="CUDA"):
        planes.append_qkv_paged(q, k, k, pool, pool, pt, pos, pos, none)
    with pytest.raises(RuntimeError):
        planes.decode_attention_shared(q, pool, pool, pt, pos)


def test_rope_tables():
    t = torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="both"):
        planes.Rope(t, None)
    with pytest.raises(RuntimeError, match="CUDA"):
        planes.Rope(t, t)


def test_structs_match_the_header():
    assert ctypes.sizeof(_lib.Heads) == 24
    assert ctypes.sizeof(_lib.Rope) == 56
