"""The 4-bit pool's operators together, as a server uses them: behind the
cache object and its drop-ins, behind block tables that grow on the device,
in the model runner and in the serving loop."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from pagedserve_b200 import (PagedKVCache, ops, paged_decode_attention, paged_decode_attention_with_write,
                             rope_and_write_tokens, write_tokens)
from pagedserve_b200.paged_kv import BlockManager
from tests import int4_reference as ref
from tests.qwen_reference import random_tables, reference_decode, reference_prefill_logits, small_qwen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    torch.backends.cuda.matmul.allow_tf32 = False


def _rand(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


# ---- the cache object and the drop-ins ------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32), (6, 3)])
def test_cache_rows_and_blocks(dtype, d, bs):
    """What write_token and write_block put in, read_token and read_block
    give back as the format's own rounding of it."""
    gen = torch.Generator().manual_seed(1)
    cache = PagedKVCache(num_blocks=6, num_layers=2, num_kv_heads=3, head_dim=d, block_size=bs, dtype=dtype,
                         kv_bits=4)
    cache.allocate("A", 2 * bs + 1)

    def want(x):
        code, step, mid = ref.quantize(x.cpu())
        return ref.values(ref.pack(code), torch.cat([step, mid], -1)).to(dtype)

    key, value = _rand(gen, 3, d, dtype=dtype), _rand(gen, 3, d, dtype=dtype)
    cache.write_token("A", 1, 2 * bs, key, value)
    k, v = cache.read_token("A", 1, 2 * bs)
    h = 2 * ref.HALF_STEP[dtype]  # one rounding on each side
    for got, x in ((k, key), (v, value)):
        torch.testing.assert_close(got.cpu().double(), want(x).double(), rtol=h, atol=2.0 ** -22)
    key, value = _rand(gen, 3, bs, d, dtype=dtype), _rand(gen, 3, bs, d, dtype=dtype)
    cache.kv_cache.write_block(0, 4, key, value)
    k, v = cache.kv_cache.read_block(0, 4)
    assert k.shape == v.shape == key.shape
    for got, x in ((k, key), (v, value)):
        torch.testing.assert_close(got.cpu().double(), want(x).double(), rtol=h, atol=2.0 ** -22)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dropins_equal_the_operators(dtype):
    """write_tokens, rope_and_write_tokens and both attention entry points on
    a 4-bit cache: the pool bytes and outputs of the operators they stand for."""
    gen = torch.Generator().manual_seed(2)
    hq, hkv, d, bs = 14, 2, 64, 16
    cache = PagedKVCache(num_blocks=90, num_layers=2, num_kv_heads=hkv, head_dim=d, block_size=bs, dtype=dtype,
                         kv_bits=4, free_order=torch.randperm(90, generator=gen).tolist())
    lens = [1, 16, 17, 300, 640]
    ids = [f"r{i}" for i in range(len(lens))]
    for r, n in zip(ids, lens):
        cache.allocate(r, n)
    kv = cache.kv_cache
    codes, params = ref.make_pool(gen, 2, 90, hkv, bs, d, dtype)
    kv.kv_codes.copy_(codes)
    kv.kv_params.copy_(params)
    codes, params = kv.kv_codes.clone(), kv.kv_params.clone()
    pos = [n - 1 for n in lens]
    b = len(lens)
    q, k, v = _rand(gen, b, hq, 1, d, dtype=dtype), _rand(gen, b, hkv, 1, d, dtype=dtype), _rand(gen, b, hkv, 1, d, dtype=dtype)
    cos, sin = _rand(gen, b, 1, d, dtype=dtype), _rand(gen, b, 1, d, dtype=dtype)
    slots = torch.tensor([cache.slot_of(r, p) for r, p in zip(ids, pos)], device="cuda")
    table = torch.from_numpy(cache.table_rows(ids)).cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def check(layer):
        assert torch.equal(kv.kv_codes, codes) and torch.equal(kv.kv_params, params)
        return ops.paged_decode_int4(q, codes, params, table, lens_t, layer)

    write_tokens(cache, ids, pos, 0, k, v)
    ops.reshape_and_cache_int4(k.squeeze(2), v.squeeze(2), codes, params, slots, 0)
    assert torch.equal(paged_decode_attention(q, cache, ids, pos, 0), check(0))
    turned = rope_and_write_tokens(q, k, v, cos, sin, cache, ids, pos, 1)
    want, _ = ops.rope_reshape_and_cache_int4(q.squeeze(2), k.squeeze(2), v.squeeze(2), cos.squeeze(1), sin.squeeze(1),
                                              codes, params, slots, 1, key_out=False)
    assert torch.equal(turned, want.unsqueeze(2))
    assert torch.equal(paged_decode_attention(q, cache, ids, pos, 1), check(1))
    for _ in range(2):  # the second call finds the first one's metadata
        k, v = _rand(gen, b, hkv, 1, d, dtype=dtype), _rand(gen, b, hkv, 1, d, dtype=dtype)
        out = paged_decode_attention_with_write(q, k, v, cache, ids, pos, 1)
        ops.reshape_and_cache_int4(k.squeeze(2), v.squeeze(2), codes, params, slots, 1)
        assert torch.equal(out, check(1))
    with pytest.raises(ValueError, match="Invalid layer"):
        paged_decode_attention(q, cache, ids, pos, 2)
    with pytest.raises(ValueError, match="Invalid position"):
        paged_decode_attention(q, cache, ids, [1] + pos[1:], 0)


# ---- a server's steps: tables, write, attention, release ---------------------------
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_serving_steps(dtype, graph):
    """Prompts in chunks, decode steps, two requests that finish and one that
    joins, with the block tables kept on the device throughout: the tables
    against BlockManager, every output against 64 bits over the rows the pool
    then holds.  ``graph``: each decode step is one replay of one capture."""
    gen = torch.Generator().manual_seed(3)
    hq, hkv, d, bs, blocks, width = 14, 2, 64, 16, 64, 24
    codes = torch.zeros(1, blocks, hkv, 2, bs, d // 2, dtype=torch.uint8, device="cuda")
    params = torch.zeros(1, blocks, hkv, 2, bs, 2, dtype=dtype, device="cuda")
    store = torch.full((6, width), -1, dtype=torch.int32, device="cuda")
    free, state = ops.free_list(blocks, "cuda")
    manager = BlockManager(blocks, bs)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    scale = d ** -0.5
    held = {}

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def grow(row, n):
        if row not in held:
            manager.allocate(str(row), n)
            held[row] = n
            return
        more = manager.blocks_needed(held[row] + n) - manager.blocks_needed(held[row])
        if more:
            manager.allocate_blocks(str(row), more)
        held[row] += n

    def check(out, q, rows, news, slots):
        at = 0
        pool = codes.cpu(), params.cpu()
        for row, n in zip(rows, news):
            blk = torch.tensor(manager.get_blocks(str(row)))
            pos = torch.arange(held[row] - n, held[row])
            assert torch.equal(slots[at:at + n].cpu(), blk[pos // bs] * bs + pos % bs)
            want, tol = ref.attend(q[at:at + n].cpu(), *pool, 0, blk, held[row], bs, held[row] - n, scale)
            assert ((out[at:at + n].cpu().double() - want).abs() <= tol).all()
            at += n

    def step(plan, starts, news, total, q, k, v, cos, sin, most):
        cu, ctx, slots, pos, tables = ops.extend_step(store, plan, starts, news, free, state, total, bs,
                                                      error_flag=err)
        qr, _ = ops.rope_reshape_and_cache_int4(q, k, v, cos.index_select(0, pos), sin.index_select(0, pos), codes,
                                                params, slots, 0, key_out=False, error_flag=err)
        if most == 1:
            out = ops.paged_decode_int4(qr, codes, params, tables, ctx, 0, error_flag=err)
        else:
            out = ops.paged_prefill_int4(qr, codes, params, tables, ctx, cu, most, 0, error_flag=err)
        return out, qr, slots

    angles = torch.arange(400)[:, None] * torch.exp(-torch.arange(0, d, 2) / d * 9)[None]
    cos = torch.cat([angles, angles], -1).cos().to(dtype).cuda()
    sin = torch.cat([angles, angles], -1).sin().to(dtype).cuda()

    def run(rows, news):
        total = sum(news)
        starts = [held.get(r, 0) for r in rows]
        for r, n in zip(rows, news):
            grow(r, n)
        q, k, v = (_rand(gen, total, h, d, dtype=dtype) for h in (hq, hkv, hkv))
        out, qr, slots = step(i32(rows), i32(starts), i32(news), total, q, k, v, cos, sin, max(news))
        check(out, qr, rows, news, slots)

    def trim(rows, keeps):
        ops.trim_tables(store, i32(rows), i32([held[r] for r in rows]), i32(keeps), free, state, bs, error_flag=err)
        for r, keep in zip(rows, keeps):
            assert keep == 0
            manager.free(str(r))
            del held[r]

    run([0, 3, 1], [40, 1, 100])
    run([3, 0, 1], [129, 7, 30])        # second chunks over what the first wrote
    trim([1], [0])
    run([4], [33])                      # joins: takes the head of the ring
    if not graph:
        for _ in range(3):
            run([0, 4, 3], [1, 1, 1])
    else:
        rows = [0, 4, 3]
        plan, starts, news = i32(rows), i32([held[r] for r in rows]), i32([1, 1, 1])
        bufs = [_rand(gen, 3, h, d, dtype=dtype) for h in (hq, hkv, hkv)]
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            got = step(plan, starts, news, 3, *bufs, cos, sin, 1)
            starts += 1
        for _ in range(20):             # each crosses a block's end at another step
            for buf in bufs:
                buf.copy_(_rand(gen, *buf.shape, dtype=dtype))
            for r in rows:
                grow(r, 1)
            g.replay()
            torch.cuda.synchronize()
            check(got[0], got[1], rows, [1, 1, 1], got[2])
        g.reset()
    trim([3, 0, 4], [0, 0, 0])
    assert err.item() == 0
    head, count = state[:2].tolist()
    ring = free.tolist()
    assert count == blocks and (ring[head:] + ring[:head]) == list(manager._free)


# ---- the model runner and the serving loop -----------------------------------------------
class _Held:
    """A pool the reference forward reads but does not write: what a 4-bit pool holds, as floats."""

    def __init__(self, values):
        self._values = values

    def __setitem__(self, index, rows):
        pass

    def float(self):
        return self._values


def _held(codes, params):
    v = ref.values(codes.cpu(), params.cpu()).float()
    return _Held(v[:, :, :, 0]), _Held(v[:, :, :, 1])


def _pool(layers, blocks, dtype, seed):
    codes, params = ref.make_pool(torch.Generator().manual_seed(seed), layers, blocks, 2, 16, 64, dtype)
    return codes.cuda(), params.cuda()


def _table(tables):
    out = torch.zeros(len(tables), max(len(t) for t in tables), dtype=torch.int32)
    for i, t in enumerate(tables):
        out[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    return out.cuda()


def test_runner_decode_matches_reference_over_the_held_rows():
    """A decode step in fp32 over a 4-bit pool against the reference forward
    whose attention reads the values that pool holds (the new token's
    included): the bound of the same step over 16-bit pools.  The rows that
    were written lie within half a step of those a pool of floats takes."""
    from pagedserve_b200.model_runner import PagedModelRunner, QwenWeights
    model = small_qwen(dtype=torch.float32, seed=21)
    rng = np.random.default_rng(21)
    lens = [1, 17, 64, 300, 1000, 2500]
    blocks = sum(-(-n // 16) for n in lens) + 7
    tables = random_tables(rng, lens, blocks)
    codes, params = _pool(2, blocks, torch.float32, 21)
    pos = [n - 1 for n in lens]
    tokens = torch.tensor(rng.integers(0, model.config.vocab_size, len(lens)), device="cuda")
    slots = torch.tensor([t[p // 16] * 16 + p % 16 for t, p in zip(tables, pos)], device="cuda")
    w = QwenWeights.from_hf(model)
    args = (tokens, torch.tensor(pos, device="cuda"), _table(tables), torch.tensor(lens, dtype=torch.int32, device="cuda"), slots)
    got = PagedModelRunner(w, codes, params, kv_bits=4).decode(*args)
    want = reference_decode(model, tokens, pos, *_held(codes, params), tables)
    assert (got - want).abs().max().item() <= 2e-4
    plain = torch.zeros(2, blocks, 2, 16, 64, device="cuda")
    kc, vc = plain, plain.clone()
    PagedModelRunner(w, kc, vc).decode(*args)
    k4, v4 = ops.gather_cache_int4(codes, params, slots, 0)
    rows = lambda c: c[0].transpose(1, 2).reshape(-1, 2, 64)[slots]
    for x4, x, i in ((k4, rows(kc), 0), (v4, rows(vc), 1)):  # layer 0: the same rows went in
        step = params[0].transpose(1, 3).reshape(-1, 2, 2, 2)[slots][:, i, :, :1]
        assert ((x4 - x).abs() <= step / 2 + 2.0 ** -20 * (x.abs().amax(-1, keepdim=True) + step)).all()


def test_runner_mixed_pass_matches_reference():
    """Prompts and decode rows in one pass over a 4-bit pool, fp32: the
    prompts' logits against the full forward (a prompt attends to its own
    unrounded rows), the decode rows' against the held values; then a decode
    step of the new prompts."""
    from pagedserve_b200.model_runner import PagedModelRunner, QwenWeights
    model = small_qwen(dtype=torch.float32, seed=22)
    rng = np.random.default_rng(22)
    plens, dlens = [3, 200, 77], [1, 40, 513, 1200]
    blocks = sum(-(-n // 16) for n in [n + 1 for n in plens] + dlens) + 4
    tables = random_tables(rng, [n + 1 for n in plens] + dlens, blocks)
    ptab, dtab = tables[:len(plens)], tables[len(plens):]
    codes, params = _pool(2, blocks, torch.float32, 22)
    runner = PagedModelRunner(QwenWeights.from_hf(model), codes, params, kv_bits=4)
    slot = lambda t, p: t[p // 16] * 16 + p % 16
    prompts = [torch.tensor(rng.integers(0, 512, n), device="cuda") for n in plens]
    dtok = torch.tensor(rng.integers(0, 512, len(dlens)), device="cuda")
    pos = torch.cat([torch.arange(n) for n in plens] + [torch.tensor([n - 1 for n in dlens])]).cuda()
    slots = torch.tensor([slot(t, p) for t, n in zip(ptab, plens) for p in range(n)]
                         + [slot(t, n - 1) for t, n in zip(dtab, dlens)], device="cuda")
    cu = torch.tensor([0] + list(np.cumsum(plens)), dtype=torch.int32, device="cuda")
    tp = sum(plens)
    last = torch.cat([(cu[1:] - 1).long(), torch.arange(tp, tp + len(dlens), device="cuda")])
    got = runner.mixed(torch.cat(prompts + [dtok]), pos, slots, tp, cu, max(plens), _table(dtab),
                       torch.tensor(dlens, dtype=torch.int32, device="cuda"), last)
    for i, p in enumerate(prompts):
        assert (got[i] - reference_prefill_logits(model, p)).abs().max().item() <= 2e-4
    want = reference_decode(model, dtok, [n - 1 for n in dlens], *_held(codes, params), dtab)
    assert (got[len(plens):] - want).abs().max().item() <= 2e-4
    nxt = got[:len(plens)].argmax(-1)
    pos = torch.tensor(plens, device="cuda")
    slots = torch.tensor([slot(t, n) for t, n in zip(ptab, plens)], device="cuda")
    got = runner.decode(nxt, pos, _table(ptab), (pos + 1).to(torch.int32), slots)
    want = reference_decode(model, nxt, plens, *_held(codes, params), ptab)
    assert (got - want).abs().max().item() <= 2e-4


def test_engine_serves_from_int4_pools():
    """The serving loop over 4-bit pools: every request runs to its budget,
    first tokens (a prompt's own pass) are the reference's, and the physical
    order of the blocks changes no token."""
    from pagedserve_b200.model_runner import QwenWeights
    from pagedserve_b200.serving import ReplicaEngine, ServeRequest
    model = small_qwen(dtype=torch.float32, seed=23)
    rng = np.random.default_rng(23)
    shapes = [(3, 5), (40, 3), (100, 18), (7, 1), (60, 6), (200, 24)]
    prompts = [rng.integers(0, 512, n) for n, _ in shapes]
    runs = []
    for order in (None, list(reversed(range(256)))):
        eng = ReplicaEngine(QwenWeights.from_hf(model), num_blocks=256, max_running=3, max_prefill_tokens=256,
                            max_prefill_seqs=2, max_prompt=256, max_context=512, decode_buckets=(2, 3),
                            prefill_buckets=(128, 256), record_tokens=True, free_order=order, kv_bits=4)
        eng.capture()
        reqs = [ServeRequest(f"r{i}", p, m) for i, (p, (_, m)) in enumerate(zip(prompts, shapes))]
        for r in reqs:
            eng.submit(r)
        done = []
        for _ in range(100):
            if not eng.has_work:
                break
            done += eng.step()
        eng.check_errors()
        eng.release()
        assert sorted(r.request_id for r in done) == sorted(r.request_id for r in reqs)
        assert eng.cache.used_blocks == -(-128 // 16)
        runs.append([r.tokens for r in reqs])
    for p, (_, m), tokens in zip(prompts, shapes, runs[0]):
        assert len(tokens) == m
        assert tokens[0] == int(reference_prefill_logits(model, torch.tensor(p, device="cuda")).argmax())
    assert runs[0] == runs[1]


def test_device_tables_feed_the_16_bit_pool():
    """extend_step, an ordinary launch, the rotary write and paged_decode over
    16-bit pools as one replayed capture whose tables change with every
    replay: the rows of a step on the host's tables."""
    gen = torch.Generator().manual_seed(11)
    hq, hkv, d, bs, blocks, width = 14, 2, 64, 16, 40, 12
    kc, vc = (torch.zeros(1, blocks, hkv, bs, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    wk, wv = kc.clone(), vc.clone()
    free, state = ops.free_list(blocks, "cuda")
    manager = BlockManager(blocks, bs)
    store = torch.zeros(4, width, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    angles = torch.arange(400)[:, None] * torch.exp(-torch.arange(0, d, 2) / d * 9)[None]
    cos = torch.cat([angles, angles], -1).cos().bfloat16().cuda()
    sin = torch.cat([angles, angles], -1).sin().bfloat16().cuda()
    rows, held = [2, 0, 3], [0, 0, 0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    plan, starts, news = i32(rows), i32(held), i32([1, 1, 1])
    q, k, v = (_rand(gen, 3, h, d) for h in (hq, hkv, hkv))
    for r in rows:
        manager.allocate(str(r), 1)
    ops.paged_decode(q, kc, vc, i32([[0] * width] * 3), i32([1] * 3), 0)  # the workspace, before the capture
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        _, ctx, slots, pos, tables = ops.extend_step(store, plan, starts, news, free, state, 3, bs, error_flag=err)
        c, s = cos.index_select(0, pos), sin.index_select(0, pos)
        qr, _ = ops.rope_reshape_and_cache(q, k, v, c, s, kc, vc, slots, 0, key_out=False)
        out = ops.paged_decode(qr, kc, vc, tables, ctx, 0)
        starts += 1
    for step in range(60):
        for buf in (q, k, v):
            buf.copy_(_rand(gen, *buf.shape))
        if step:
            for r in rows:
                if manager.blocks_needed(step + 1) > manager.blocks_needed(step):
                    manager.allocate_blocks(str(r), 1)
        g.replay()
        ids = [manager.get_blocks(str(r)) for r in rows]
        tab = i32([b + [0] * (width - len(b)) for b in ids])
        slot = torch.tensor([b[step // bs] * bs + step % bs for b in ids], device="cuda")
        at = torch.full((3,), step, device="cuda")
        wq, _ = ops.rope_reshape_and_cache(q, k, v, cos.index_select(0, at), sin.index_select(0, at), wk, wv, slot, 0,
                                           key_out=False)
        torch.cuda.synchronize()
        want = ops.paged_decode(wq, wk, wv, tab, i32([step + 1] * 3), 0)
        assert torch.equal(out, want) and torch.equal(kc, wk) and torch.equal(vc, wv)
    assert err.item() == 0
    g.reset()


@pytest.mark.parametrize("d", [64, 6])
def test_cache_takes_rows_of_any_strides(d):
    """Rows whose elements are not adjacent go into a 4-bit cache as they do
    into a 16-bit one, by token, by block and in the fused decode call."""
    gen = torch.Generator().manual_seed(12)
    bs, hkv = 4, 2
    caches = [PagedKVCache(num_blocks=6, num_layers=1, num_kv_heads=hkv, head_dim=d, block_size=bs,
                           dtype=torch.bfloat16, kv_bits=4) for _ in range(2)]
    for c in caches:
        c.allocate("A", 6)
        c.kv_cache.kv_codes.zero_()
        c.kv_cache.kv_params.zero_()

    def strided(t):
        wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
        wide[..., 0] = t
        return wide[..., 0]

    token = [_rand(gen, hkv, d) for _ in range(2)]
    block = [_rand(gen, hkv, bs, d) for _ in range(2)]
    new = [_rand(gen, 1, hkv, 1, d) for _ in range(2)]
    q = _rand(gen, 1, 4, 1, d)
    outs = []
    for c, view in zip(caches, (lambda t: t, strided)):
        for pos in range(5):
            c.write_token("A", 0, pos, *(view(t) for t in token))
        c.kv_cache.write_block(0, 5, *(view(t) for t in block))
        outs.append(paged_decode_attention_with_write(view(q), view(new[0]), view(new[1]), c, ["A"], [5], 0))
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(caches[0].kv_cache.kv_codes, caches[1].kv_cache.kv_codes)
    assert torch.equal(caches[0].kv_cache.kv_params, caches[1].kv_cache.kv_params)
