"""Refusals of the calls for shared pages, shared prefixes and verified drafts, on the CPU: what the arguments alone show."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pagedserve_b200 import _native, ops

I32 = torch.int32


def _i32(v):
    return torch.tensor(v, dtype=I32)


def _pages(**kw):
    a = dict(table_store=torch.zeros(6, 8, dtype=I32), first=_i32([0, 0]), second=_i32([1, 2]), third=_i32([5, 5]),
             shares=torch.zeros(2, 20, dtype=I32), free=torch.arange(20, dtype=I32), state=_i32([0, 20, 0, 0]), bs=16)
    a.update(kw)
    return a.values()


BAD_PAGES = [
    (dict(table_store=torch.zeros(6, 8)), "table_store"), (dict(table_store=torch.zeros(8, 6, dtype=I32).t()), "table_store"),
    (dict(first=_i32([0])), "int32 \\[B\\]"), (dict(second=torch.zeros(2, dtype=torch.int64)), "int32 \\[B\\]"),
    (dict(free=torch.zeros(0, dtype=I32)), "free_blocks"), (dict(state=_i32([0, 1])), "free_state"), (dict(bs=0), "block_size"),
    (dict(shares=torch.zeros(2, 19, dtype=I32)), "shares"), (dict(shares=torch.zeros(20, dtype=I32)), "shares"),
    (dict(shares=torch.zeros(20, 2, dtype=I32).t()), "shares"), (dict(shares=torch.zeros(2, 20)), "shares"), ({}, "CUDA")]


@pytest.mark.parametrize("call", [ops.fork_tables, ops.release_tables])
@pytest.mark.parametrize("kw,text", BAD_PAGES, ids=range(len(BAD_PAGES)))
def test_page_calls_refuse(call, kw, text):
    with pytest.raises(ValueError, match=text):
        call(*_pages(**kw))
    with pytest.raises(ValueError, match="error_flag"):
        call(*_pages(), error_flag=torch.zeros(1))


def test_share_counts():
    assert ops.share_counts(5, "cpu").shape == (2, 5) and not ops.share_counts(5, "cpu").any()
    with pytest.raises(ValueError):
        ops.share_counts(0, "cpu")


@pytest.mark.parametrize("pools,src,dst,text", [
    ((), _i32([1]), _i32([2]), "one to four"), ((torch.zeros(1, 2, 3),) * 5, _i32([1]), _i32([0]), "one to four"),
    ((torch.zeros(1, 2, 3),), _i32([1]), _i32([0, 1]), "int32 \\[N\\]"), ((torch.zeros(1, 2, 3),), torch.zeros(1), torch.zeros(1), "int32 \\[N\\]"),
    ((torch.zeros(1, 2, 3), torch.zeros(1, 3, 3)), _i32([1]), _i32([0]), "contiguous"), ((torch.zeros(1, 2),), _i32([1]), _i32([0]), "contiguous"),
    ((torch.zeros(2, 3, 3).transpose(0, 1),), _i32([1]), _i32([0]), "contiguous"), ((torch.zeros(1, 2, 3),), _i32([1]), _i32([0]), "CUDA")])
def test_copy_blocks_refuses(pools, src, dst, text):
    with pytest.raises(ValueError, match=text):
        ops.copy_blocks(pools, src, dst)


def _shared(**kw):
    pool = torch.zeros(2, 9, 2, 16, 64, dtype=torch.bfloat16)
    a = dict(query=torch.zeros(3, 14, 64, dtype=torch.bfloat16), k=pool, v=pool, table=torch.zeros(3, 4, dtype=I32), lens=_i32([5, 6, 7]),
             cu=_i32([0, 2]), prefix=_i32([3]), layer=0)
    opt = {k: kw.pop(k) for k in list(kw) if k not in a}
    a.update(kw)
    return list(a.values()), opt


BAD_SHARED = [
    (dict(query=torch.zeros(3, 14, 32, dtype=torch.bfloat16)), "query"), (dict(query=torch.zeros(3, 15, 64, dtype=torch.bfloat16)), "divisible"),
    (dict(query=torch.zeros(3, 14, 64)), "dtype"), (dict(query=torch.zeros(0, 14, 64, dtype=torch.bfloat16)), "empty"),
    (dict(query=torch.zeros(3, 14, 2, 64, dtype=torch.bfloat16)), "query"), (dict(v=torch.zeros(2, 9, 2, 16, 32, dtype=torch.bfloat16)), "k_cache"),
    (dict(table=torch.zeros(2, 4, dtype=I32)), "block_tables"), (dict(table=torch.zeros(3, 4)), "block_tables"), (dict(lens=_i32([1, 2])), "context_lens"),
    (dict(cu=_i32([0])), "cu_groups"), (dict(cu=torch.zeros(2, dtype=torch.int64)), "cu_groups"), (dict(prefix=torch.zeros(1)), "prefix_lens"),
    (dict(layer=2), "layer"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(max_context=65), "max_context"), (dict(max_context=-1), "max_context"),
    (dict(out=torch.zeros(3, 14, 64)), "out"), (dict(out=torch.zeros(3, 14, 128, dtype=torch.bfloat16)[..., ::2]), "out"),
    (dict(error_flag=torch.zeros(1)), "error_flag"), ({}, "CUDA")]


@pytest.mark.parametrize("kw,text", BAD_SHARED, ids=range(len(BAD_SHARED)))
def test_paged_decode_shared_refuses(kw, text):
    args, opt = _shared(**kw)
    with pytest.raises(ValueError, match=text):
        ops.paged_decode_shared(*args, **opt)


def test_which_geometries_share():
    f = ops.decode_shared_workspace_bytes
    assert f(64, 1, 14, 2, 64, 16, 4096, torch.bfloat16) > 0 and f(64, 64, 32, 8, 128, 128, 4096, torch.float16) > 0
    assert f(2048, 2048, 16, 1, 64, 64, 1 << 20, torch.bfloat16) > 0
    for other in ((64, 1, 14, 2, 64, 16, 4096, torch.float32), (64, 1, 14, 2, 96, 16, 4096, torch.bfloat16), (64, 1, 14, 2, 64, 8, 4096, torch.bfloat16),
                  (64, 1, 14, 2, 64, 48, 4096, torch.bfloat16), (64, 1, 34, 2, 64, 16, 4096, torch.bfloat16), (2049, 1, 14, 2, 64, 16, 4096, torch.bfloat16),
                  (64, 2049, 14, 2, 64, 16, 4096, torch.bfloat16), (64, 1, 15, 2, 64, 16, 4096, torch.bfloat16), (0, 0, 14, 2, 64, 16, 4096, torch.bfloat16)):
        assert f(*other) == 0


def _verify(**kw):
    a = dict(logits=torch.zeros(5, 30), tokens=torch.zeros(5, dtype=torch.int64), cu=_i32([0, 2, 5]), uniforms=torch.zeros(5, 2), temperature=torch.ones(2))
    opt = {k: kw.pop(k) for k in list(kw) if k not in a}
    a.update(kw)
    return list(a.values()), opt


BAD_VERIFY = [
    (dict(logits=torch.zeros(5)), "logits"), (dict(logits=torch.zeros(5, 0)), "logits"), (dict(logits=torch.zeros(5, 30, dtype=torch.float64)), "dtype"),
    (dict(tokens=torch.zeros(5, dtype=I32)), "tokens"), (dict(tokens=torch.zeros(4, dtype=torch.int64)), "tokens"), (dict(cu=torch.zeros(3)), "cu_seqlens"),
    (dict(cu=torch.zeros(0, dtype=I32)), "cu_seqlens"), (dict(cu=_i32([0]), temperature=torch.ones(0)), "no sequence"), (dict(uniforms=torch.zeros(5)), "uniforms"),
    (dict(uniforms=torch.zeros(5, 2, dtype=torch.float64)), "uniforms"), (dict(temperature=torch.ones(3)), "temperature"),
    (dict(draft_probs=torch.zeros(5, 29)), "draft_probs"), (dict(draft_probs=torch.zeros(5, 30, dtype=torch.int32)), "dtype"),
    (dict(out=(torch.zeros(5, dtype=torch.int64), torch.zeros(2))), "out"), (dict(error_flag=torch.zeros(1)), "error_flag"), ({}, "CUDA")]


@pytest.mark.parametrize("kw,text", BAD_VERIFY, ids=range(len(BAD_VERIFY)))
def test_verify_tokens_refuses(kw, text):
    args, opt = _verify(**kw)
    with pytest.raises(ValueError, match=text):
        ops.verify_tokens(*args, **opt)


def test_verify_tokens_does_not_write_over_its_drafts():
    args, _ = _verify()
    with pytest.raises(ValueError, match="itself"):
        ops.verify_tokens(*args, out=(args[1], torch.zeros(2, dtype=I32)))


def test_c_entries_refuse_without_a_gpu():
    lib = _native.load()
    inv, ws, unsup = _native.PSB_ERR_INVALID, _native.PSB_ERR_WORKSPACE, _native.PSB_ERR_UNSUPPORTED
    p = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p).value + 4095 & ~4095 & -16
    fork = lambda **kw: lib.psb_fork_tables(*{**dict(store=p, stride=8, rows=6, width=8, a=p, b=p, c=p, batch=2, shares=p, ring=p, n=20, state=p, bs=16,
                                                     src=p, dst=p, err=None, s=None), **kw}.values())
    release = lambda **kw: lib.psb_release_tables(*{**dict(store=p, stride=8, rows=6, width=8, a=p, b=p, c=p, batch=2, shares=p, ring=p, n=20, state=p,
                                                           bs=16, err=None, s=None), **kw}.values())
    for call in (fork, release):
        for kw in (dict(batch=-1), dict(bs=0), dict(rows=0), dict(stride=7), dict(n=0), dict(store=None), dict(shares=None), dict(a=None)):
            assert call(**kw) == inv
        assert call(batch=0) == 0
    assert fork(src=None) == inv
    assert lib.psb_copy_blocks(None, None, 5, p, p, 1, 1, 1, None, None) == inv
    assert lib.psb_copy_blocks(None, None, 1, p, p, 1, 1, 1, None, None) == inv
    assert lib.psb_copy_blocks(None, None, 1, p, p, 0, 1, 1, None, None) == 0
    dec = lambda **kw: lib.psb_paged_decode_shared(*{**dict(q=p, qb=896, qh=64, o=p, ob=896, oh=64, k=p, v=p, t=p, ts=4, ctx=p, cu=p, pre=p, batch=2, groups=1,
                                                            hq=14, layer=0, layers=1, blocks=9, hkv=2, bs=16, d=64, dt=2, most=64, scale=0.1, ws=None,
                                                            wsn=0, err=None, s=None), **kw}.values())
    for kw in (dict(batch=-1), dict(hq=15), dict(layer=1), dict(blocks=0), dict(scale=0.0), dict(scale=float("nan")), dict(dt=7), dict(q=None), dict(cu=None)):
        assert dec(**kw) == inv
    for kw in (dict(dt=0), dict(d=96), dict(bs=8), dict(qb=895), dict(q=p + 2), dict(qb=0)):
        assert dec(**kw) == unsup
    assert dec() == ws and dec(ws=p, wsn=64) == ws and dec(batch=0) == 0
    ver = lambda **kw: lib.psb_verify_tokens(*{**dict(x=p, rs=30, t=5, v=30, dt=0, tok=p, cu=p, b=2, u=p, heat=p, q=None, qs=0, qd=0, out=p, n=p, ws=p,
                                                      wsn=64, err=None, s=None), **kw}.values())
    for kw in (dict(t=-1), dict(v=0), dict(b=-1), dict(rs=29), dict(dt=9), dict(q=p, qs=29), dict(q=p, qs=30, qd=9), dict(b=0), dict(x=None), dict(heat=None),
               dict(x=p + 1), dict(out=None)):
        assert ver(**kw) == inv
    assert ver(t=0, b=0) == 0
    assert ver(ws=None) == ws and ver(ws=p + 8) == ws and ver(wsn=31) == ws and lib.psb_verify_tokens_workspace_size(2) == 32
