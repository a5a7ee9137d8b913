"""One prompt continued in several ways: forked pages, attention over the shared
prefix, sampled tokens, verified drafts and pages given back, run together."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.qwen_reference import reference_decode, small_qwen
from tests.test_gpu_verify_tokens import _rule

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")
    import pagedserve_b200._native as native
    native.load()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Serving:
    """A pool, its tables and ring on the device; what each row holds, on the host in 64 bits."""

    def __init__(self, hq, hkv, d, bs, blocks, rows, width, dtype, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.bs, self.dtype = hq, hkv, d, bs, dtype
        from pagedserve_b200 import ops
        self.ops = ops
        self.store = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(blocks, generator=self.g).int().cuda()
        self.state = _i32([0, blocks, 0, 0])
        self.shares = ops.share_counts(blocks, "cuda")
        self.err = _i32([0])
        self.k = torch.full((1, blocks, hkv, bs, d), math.nan, dtype=dtype, device="cuda")
        self.v = self.k.clone()
        self.rows = {}  # row -> (keys, values) [n, hkv, d], float64

    def args(self):
        return dict(shares=self.shares, free_blocks=self.ring, free_state=self.state, block_size=self.bs, error_flag=self.err)

    def fed(self, rows, counts):
        """Steps ``rows`` on by ``counts`` tokens of random keys and values; the plan of the step."""
        starts = [len(self.rows[r][0]) if r in self.rows else 0 for r in rows]
        total = sum(counts)
        cu, ctx, slots, _, tables = self.ops.extend_step(self.store, _i32(rows), _i32(starts), _i32(counts), self.ring, self.state,
                                                         total, self.bs, error_flag=self.err)
        key, value = (torch.randn(total, self.hkv, self.d, generator=self.g).to(self.dtype) for _ in range(2))
        self.ops.reshape_and_cache(key.cuda(), value.cuda(), self.k, self.v, slots, 0, error_flag=self.err)
        at = 0
        for r, n in zip(rows, counts):
            old = self.rows.get(r, (torch.zeros(0, self.hkv, self.d, dtype=torch.float64),) * 2)
            self.rows[r] = tuple(torch.cat([o, x[at:at + n].double()]) for o, x in zip(old, (key, value)))
            at += n
        return cu, ctx, tables

    def keep(self, r, n):
        self.rows[r] = tuple(x[:n] for x in self.rows[r])

    def attention(self, q, rows):
        """(output, tolerance): each row's query over all that it holds."""
        half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[self.dtype]
        group = self.hq // self.hkv
        out, tol = (torch.zeros(len(rows), self.hq, self.d, dtype=torch.float64) for _ in range(2))
        for i, r in enumerate(rows):
            for h in range(self.hq):
                k, v = (x[:, h // group] for x in self.rows[r])
                qq = q[i, h].double()
                p = torch.softmax(k @ qq * self.d ** -0.5, 0)
                out[i, h] = p @ v
                # scores: d products and sums in fp32, which a probability is off by twice; its exponential, the sums
                # and the joins (2^-19 together) and its rounding; the result's rounding; f16 probabilities
                # below 2^-14 are off by 2^-25
                ds = (self.d + 4) * 2.0 ** -24 * (k.abs() @ qq.abs()).max() * self.d ** -0.5
                tiny = len(p) * 2.0 ** -25 * v.abs().max() if self.dtype == torch.float16 else 0.0
                tol[i, h] = (half * 1.01 + 2 * ds + 2.0 ** -19) * (p @ v.abs()) + half * out[i, h].abs() + tiny + 1e-9
        return out, tol


@pytest.mark.parametrize("hq,hkv,d,bs,prompts,each,dtype", [
    (14, 2, 64, 16, (37, 64), 3, torch.bfloat16),
    (8, 2, 128, 32, (129, 31, 5), 2, torch.float16),
    (4, 1, 64, 64, (700,), 6, torch.bfloat16),
])
def test_a_prompt_sampled_several_times(hq, hkv, d, bs, prompts, each, dtype):
    """Prompts are forked into several rows and their own rows given back; then steps
    of one token (attention over the shared prefix, a sample) and of several (drafts, of
    which some are taken and the rest's pages given back), until all is released."""
    blocks, vocab = 160, 1000
    s = Serving(hq, hkv, d, bs, blocks, 40, 40, dtype, seed=len(prompts))
    parents = list(range(len(prompts)))
    s.fed(parents, list(prompts))
    children = [len(prompts) + i for i in range(len(prompts) * each)]
    of = [c // each for c in range(len(children))]
    src, dst = s.ops.fork_tables(s.store, _i32([parents[p] for p in of]), _i32(children), _i32([prompts[p] for p in of]), **s.args())
    s.ops.copy_blocks((s.k, s.v), src, dst, error_flag=s.err)
    assert ((src >= 0).cpu() == torch.tensor([prompts[p] % bs != 0 for p in of])).all()
    for c, p in zip(children, of):
        s.rows[c] = s.rows[parents[p]]
    s.ops.release_tables(s.store, _i32(parents), _i32(list(prompts)), _i32([0] * len(parents)), **s.args())
    cu_groups = _i32([each * i for i in range(len(prompts) + 1)])
    heat = torch.tensor([0.0 if i % 3 == 0 else 0.7 for i in range(len(children))])
    w = torch.randn(hq * d, vocab, generator=s.g)
    last = torch.randint(0, vocab, (len(children),), generator=s.g)
    for step in range(9):
        drafts = 3 if step % 3 == 2 else 0
        cu, ctx, tables = s.fed(children, [1 + drafts] * len(children))
        t = len(children) * (1 + drafts)
        q = torch.randn(t, hq, d, generator=s.g).to(dtype)
        tokens = torch.randint(0, vocab, (t,), generator=s.g)
        tokens[::1 + drafts] = last
        u = torch.rand(t, 2, generator=s.g)
        if drafts:  # the rows of a step with drafts: no attention of one token a row; what matters is what is taken
            logits = (torch.randn(t, vocab, generator=s.g) * 4).to(dtype).cuda()
            likely = torch.cat([tokens[:1], logits.argmax(1).cpu()[:-1]])
            tokens = torch.where(torch.rand(t, generator=s.g) < 0.6, likely, tokens)
            tokens[::1 + drafts] = last
        else:
            got = s.ops.paged_decode_shared(q.cuda(), s.k, s.v, tables, ctx, cu_groups, _i32(list(prompts)), 0, error_flag=s.err)
            want, tol = s.attention(q, children)
            assert ((got.cpu().double() - want).abs() <= tol).all(), step
            logits = (got.float().reshape(len(children), -1) @ w.cuda()).to(dtype)
        new, counts = s.ops.verify_tokens(logits, tokens.cuda(), cu, u.cuda(), heat.cuda(), error_flag=s.err)
        want, n = _rule(logits.cpu(), tokens, cu.tolist(), u, heat, None)
        assert torch.equal(new.cpu(), want) and torch.equal(counts.cpu(), n), step
        last = torch.stack([new.cpu()[a + c - 1] for a, c in zip(cu.tolist(), counts.tolist())])
        if drafts:  # the rows of drafts that were not taken go back (their pages, where those are empty)
            s.ops.release_tables(s.store, _i32(children), ctx, ctx - (1 + drafts) + counts, **s.args())
            for r, c in zip(children, counts.tolist()):
                s.keep(r, len(s.rows[r][0]) - (1 + drafts) + c)
    held = [len(s.rows[c][0]) for c in children]
    s.ops.release_tables(s.store, _i32(children), _i32(held), _i32([0] * len(children)), **s.args())
    assert int(s.err) == 0
    assert s.state.tolist()[1] == blocks and int(s.shares.abs().sum()) == 0
    head = int(s.state[0])
    assert sorted(s.ring.tolist()) == list(range(blocks)) and 0 <= head < blocks


def test_a_model_decodes_forked_requests():
    """A decode step of PagedModelRunner over requests forked from one prompt in a
    PagedKVCache, with their shared prefixes named, against transformers' modules and the
    oracle's attention, at the tolerances of the plain decode step's bf16 test."""
    from pagedserve_b200 import PagedKVCache
    from pagedserve_b200.model_runner import PagedModelRunner, QwenWeights
    model = small_qwen(dtype=torch.bfloat16, seed=5)
    cache = PagedKVCache(600, 2, 2, 64, device="cuda")
    for pool in (cache.kv_cache.k_cache, cache.kv_cache.v_cache):
        pool.copy_(torch.randn(pool.shape, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda"))
    cache.allocate("p", 1000)
    cache.allocate("alone", 77)
    cache.fork("p", ["a", "b", "c"])
    cache.append_tokens("b", 40)
    cache.append_tokens("c", 200)
    cache.fork("c", ["d"], 1100)
    ids = ["p", "a", "b", "c", "d", "alone"]
    for r in ids:
        cache.append_tokens(r, 1)
    lens = [cache.token_count(r) for r in ids]
    tables = [cache.get_block_table(r).get_blocks() for r in ids]
    kc, vc = cache.kv_cache.k_cache, cache.kv_cache.v_cache
    for name in ("a", "b", "c"):  # the fork's copy of the unfinished block
        a, b = cache.get_block_table("p").get_blocks()[62], cache.get_block_table(name).get_blocks()[62]
        assert a != b and torch.equal(kc[:, a], kc[:, b]) and torch.equal(vc[:, a], vc[:, b])
    kc_ref, vc_ref = kc.clone(), vc.clone()
    positions = [n - 1 for n in lens]
    tokens = torch.tensor(np.random.default_rng(5).integers(0, model.config.vocab_size, len(ids)), device="cuda")
    want = reference_decode(model, tokens, positions, kc_ref, vc_ref, tables)
    runner = PagedModelRunner(QwenWeights.from_hf(model), kc, vc)
    cu, prefix = cache.shared_prefixes(ids)
    assert cu.tolist() == [0, 5, 6] and prefix.tolist() == [62 * 16, 0]
    slots = torch.tensor([cache.slot_of(r, n - 1) for r, n in zip(ids, lens)], device="cuda")
    got = runner.decode(tokens, torch.tensor(positions, device="cuda"), torch.from_numpy(cache.table_rows(ids)).cuda(), _i32(lens), slots,
                        groups=(torch.from_numpy(cu).cuda(), torch.from_numpy(prefix).cuda()))
    diff = (got.float() - want.float()).abs()
    assert diff.max().item() <= 6e-2 and diff.mean().item() <= 6e-3, (diff.max().item(), diff.mean().item())
    for a, b in ((kc, kc_ref), (vc, vc_ref)):
        torch.testing.assert_close(a.float(), b.float(), rtol=1.6e-2, atol=1.6e-2)


def test_four_bit_pools_fork_but_name_no_groups():
    from pagedserve_b200 import PagedKVCache
    from pagedserve_b200.model_runner import PagedModelRunner, QwenWeights
    model = small_qwen(dtype=torch.bfloat16, seed=5)
    cache = PagedKVCache(20, 2, 2, 64, device="cuda", kv_bits=4)
    kv = cache.kv_cache
    kv.kv_codes.random_(0, 256)
    kv.kv_params.normal_()
    cache.allocate("p", 21)
    cache.fork("p", ["a", "b"])
    src = cache.get_block_table("p").get_blocks()[1]
    for r in ("a", "b"):
        t = cache.get_block_table(r).get_blocks()
        assert t[0] == cache.get_block_table("p").get_blocks()[0] and t[1] != src
        assert torch.equal(kv.kv_codes[:, t[1]], kv.kv_codes[:, src])
        assert torch.equal(kv.kv_params[:, t[1]].view(torch.int16), kv.kv_params[:, src].view(torch.int16))
    runner = PagedModelRunner(QwenWeights.from_hf(model), kv.kv_codes, kv.kv_params, kv_bits=4)
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="16-bit pool"):
        runner.decode(z, z, _i32([[0]]), _i32([1]), z, groups=(_i32([0, 1]), _i32([0])))
