"""What is measured of the 4-bit paged KV cache and of the block tables built on the GPU.

Four kinds of case, one pass each:

* ``tables``   one engine step's block tables: ``ops.extend_step`` takes the blocks the step's new tokens need
               from the device free list and builds cu_seqlens, lengths, slots, positions and tables;
               ``ops.trim_tables`` then gives back what the requests do not keep;
* ``write``    new tokens' keys and values into the 4-bit pool (with or without the rotary embedding), and the
               same slots read back as the values the codes stand for;
* ``decode``   one query token per sequence over the 4-bit pool;
* ``prefill``  packed chunks of query tokens over the 4-bit pool, causal at the end of each sequence's context.

The cache format: per (token, kv head) row x of ``D`` values of type T, one offset and one step of type T,
    mid = T(lo / 2 + hi / 2),  step = T(max(hi - mid, mid - lo) / 7.5),
    code = clamp(floor((x - mid) / step) + 8, 0, 15)  (8 where step is 0),  value = mid + step (code - 7.5),
every operation before a rounding to T in float32.  ``kv_codes`` uint8 [L, NB, Hkv, 2 (K | V), BS, D / 2] holds two
codes a byte (even element low), ``kv_params`` T [L, NB, Hkv, 2, BS, 2] holds (step, mid).
"""

import math
import random

import torch

own = False

_T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# --------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a served batch of single tokens, every request one token on: the step's tables in a captured decode step
        dict(name="tables decode 256", kind="tables", batch=256, new="one", longest=4096, store=2048, block=16),
        # admission: ragged prompts of a packed prefill, tables grown from nothing or from a kept prefix
        dict(name="tables prompts 48", kind="tables", batch=48, new="ragged", longest=2000, store=2048, block=16),
        # the new tokens of a decode step
        dict(name="write step 256", kind="write", tokens=256, hq=14, hkv=2, dim=64, block=16, dtype="bf16", rope=True, keep_key=False, pad=0),
        # a full packed prefill, its keys also wanted by the attention over the fresh rows
        dict(name="write pack 16384", kind="write", tokens=16384, hq=14, hkv=2, dim=64, block=16, dtype="bf16", rope=True, keep_key=True, pad=37),
        # keys already rotated, an odd token count, padding rows, wide heads in half precision
        dict(name="write plain 1333 f16", kind="write", tokens=1333, hq=32, hkv=8, dim=128, block=32, dtype="f16", rope=False, keep_key=False, pad=5),
        # one user's next token on a short context: latency
        dict(name="decode 1 x 77", kind="decode", batch=1, hq=14, hkv=2, dim=64, block=16, dtype="bf16", lens="equal", longest=77, empty=0),
        # the served batch: 256 sequences, lengths lognormal about 1024, two idle rows
        dict(name="decode 256 x 1k", kind="decode", batch=256, hq=14, hkv=2, dim=64, block=16, dtype="bf16", lens="lognormal", longest=8192, empty=2),
        # few sequences at the longest positions: the split along the context
        dict(name="decode 3 x 32k f16", kind="decode", batch=3, hq=14, hkv=2, dim=64, block=16, dtype="f16", lens="equal", longest=32767, empty=0),
        # wide heads, groups of four, larger blocks
        dict(name="decode 64 x 4k d128", kind="decode", batch=64, hq=32, hkv=8, dim=128, block=32, dtype="bf16", lens="uniform", longest=4096, empty=1),
        # a few drafted tokens per sequence, checked in one pass
        dict(name="prefill verify 32 x 5", kind="prefill", batch=32, hq=14, hkv=2, dim=64, block=16, dtype="bf16", new=5, ragged=False, longest=1500),
        # a prompt's next chunk on a long prefix
        dict(name="prefill chunk 512 on 8k", kind="prefill", batch=1, hq=14, hkv=2, dim=64, block=16, dtype="bf16", new=512, ragged=False, longest=8192),
        # ragged chunks of several requests, in half precision
        dict(name="prefill chunks 6 x 1k f16", kind="prefill", batch=6, hq=14, hkv=2, dim=64, block=16, dtype="f16", new=1024, ragged=True, longest=6000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["tables", "write", "decode", "decode", "prefill", "prefill"])
    block = rng.choice([16, 16, 32])
    if kind == "tables":
        new = rng.choice(["one", "ragged"])
        batch = _log(rng, 1, 256) if new == "one" else _log(rng, 1, 48)
        return dict(kind=kind, batch=batch, new=new, longest=_log(rng, 16, 4000 if new == "one" else 2000), store=2048, block=block)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    hq, hkv, dim = rng.choice([(14, 2, 64), (14, 2, 64), (8, 8, 64), (12, 2, 64), (16, 1, 64), (32, 8, 128), (28, 4, 128), (10, 5, 64)])
    if kind == "write":
        tokens = _log(rng, 1, 8000)
        return dict(kind=kind, tokens=tokens, hq=hq, hkv=hkv, dim=dim, block=block, dtype=rng.choice([dtype, dtype, "f32"]), rope=rng.random() < 0.7,
                    keep_key=rng.random() < 0.5, pad=rng.randrange(0, 1 + min(tokens - 1, 40)))
    if kind == "decode":
        batch = _log(rng, 1, 200)
        cap = max(2, min(32767, 500000 // (batch * hkv * dim // 64)))
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, dim=dim, block=block, dtype=dtype, lens=rng.choice(["equal", "uniform", "lognormal"]),
                    longest=_log(rng, 1, cap), empty=rng.randrange(0, 1 + min(2, batch - 1)))
    hq, hkv, dim = rng.choice([(14, 2, 64), (14, 2, 64), (8, 8, 64), (12, 2, 64), (16, 1, 64), (10, 5, 64)])
    batch = _log(rng, 1, 24)
    new = _log(rng, 1, max(1, min(1000, 4000 // batch)))
    room = 14 * 6 * 1024 * 6000 // (batch * new * hq)
    longest = max(new, _log(rng, 1, max(2, min(8000, room))))
    return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, dim=dim, block=16, dtype=dtype, new=new, ragged=rng.random() < 0.6, longest=longest)


def _lengths(case, seed):
    """The sequences' context lengths of a decode case, longest first is not assumed."""
    r = random.Random(seed * 7 + 1)
    top, batch = case["longest"], case["batch"]
    if case["lens"] == "equal":
        lens = [max(1, top - r.randrange(0, 1 + top // 50)) for _ in range(batch)]
    elif case["lens"] == "uniform":
        lens = [r.randint(1, top) for _ in range(batch)]
    else:
        lens = [min(top, max(1, int(r.lognormvariate(math.log(max(1, top / 8)), 1.0)))) for _ in range(batch)]
    idle = {(i * 97 + 1) % batch for i in range(case["empty"])}
    return [0 if i in idle else n for i, n in enumerate(lens)]


def _parts(case, top, ragged, r):
    """``batch`` counts of new tokens up to ``top``: a case's own, in an order of the seed's."""
    own_r = random.Random(case["batch"] * 1009 + top)
    new = [own_r.randint(1, top) if ragged else top for _ in range(case["batch"])]
    r.shuffle(new)
    return new


def _chunks(case, seed):
    """(new tokens, context lengths) of a prefill case."""
    r = random.Random(seed * 7 + 2)
    new = _parts(case, case["new"], case["ragged"], r)
    ctx = [max(n, case["longest"] - r.randrange(0, 1 + (case["longest"] // 2 if case["ragged"] or case["batch"] > 1 else 16))) for n in new]
    return new, ctx


def _plan(case, seed):
    """(starts, new tokens) of a tables case."""
    r = random.Random(seed * 7 + 3)
    if case["new"] == "one":
        return [r.randrange(0, case["longest"]) for _ in range(case["batch"])], [1] * case["batch"]
    new = _parts(case, case["longest"], True, r)
    return [r.choice([0, 0, r.randrange(0, case["longest"])]) for _ in range(case["batch"])], new


def work(case):
    if case["kind"] == "tables":
        starts, new = _plan(case, 0)
        total, batch, bs = sum(new), case["batch"], case["block"]
        width = -(-2 * case["longest"] // bs)
        grown = sum(-(-(s + n) // bs) - -(-s // bs) for s, n in zip(starts, new))
        held = sum(-(-s // bs) for s in starts)
        # plan in; lengths, slots, positions, tables out; held blocks read, grown ones taken, written and given back
        return dict(bytes=4 * (3 * batch + 2 * batch + 1) + 16 * total + 4 * batch * width + 4 * held + 20 * grown, flops=0)
    hq, hkv, dim, e = case["hq"], case["hkv"], case["dim"], _SIZE[case["dtype"]]
    row = dim + 4 * e  # K and V codes of one (token, kv head) and their steps and offsets
    if case["kind"] == "write":
        t = case["tokens"]
        rot = t * dim * e * ((2 * hq + 2 + (hkv if case["keep_key"] else 0)) if case["rope"] else 0)
        live = t - case["pad"]
        return dict(bytes=rot + 2 * t * hkv * dim * e + live * hkv * row + 2 * t * hkv * dim * e + 8 * t, flops=t * dim * (3 * (hq + hkv) * case["rope"] + 12 * hkv))
    if case["kind"] == "decode":
        n = sum(_lengths(case, 0))
        return dict(bytes=n * hkv * row + 2 * case["batch"] * hq * dim * e + 4 * n // case["block"], flops=4 * hq * dim * n)
    new, ctx = _chunks(case, 0)
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, ctx))
    return dict(bytes=sum(ctx) * hkv * row + 2 * sum(new) * hq * dim * e + 4 * sum(ctx) // case["block"], flops=4 * hq * dim * pairs)


# --------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------
def _tables(lens, block, spare, generator):
    """A shuffled pool's block table for each length, zero padded, and the pool's size."""
    need = torch.tensor([-(-n // block) for n in lens])
    blocks = int(need.sum()) + spare
    have = torch.arange(max(1, int(need.max())))[None, :] < need[:, None]
    table = torch.zeros(have.shape, dtype=torch.int32)
    table[have] = torch.randperm(blocks, generator=generator)[:blocks - spare].to(torch.int32)
    return table.cuda(), blocks


def _pool(layers, blocks, case, g):
    """A 4-bit pool of normal keys and values; what no sequence reaches holds the rows of earlier requests."""
    shape = (layers, blocks, case["hkv"], 2, case["block"])
    x = torch.empty(shape + (case["dim"],), device="cuda", dtype=_T[case["dtype"]]).normal_(0, 1, generator=g)
    # a channel that stands out in the keys, as biased key projections give
    x[..., 0, :, 5] += 4.0
    codes, params = _quantize(x)
    return codes, params


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 13 + 5)
    h = torch.Generator()
    h.manual_seed(seed * 17 + 7)
    s = dict(case)
    if case["kind"] == "tables":
        starts, new = _plan(case, seed)
        bs, batch = case["block"], case["batch"]
        width = -(-2 * case["longest"] // bs)
        held = [-(-n // bs) for n in starts]
        blocks = batch * width + 300
        perm = torch.randperm(blocks, generator=h).to(torch.int32)
        rows = torch.randperm(case["store"], generator=h)[:batch].to(torch.int32)
        store = torch.zeros(case["store"], width, dtype=torch.int32)
        at = sum(held)
        have = torch.arange(width)[None, :] < torch.tensor(held)[:, None]
        table = torch.zeros(batch, width, dtype=torch.int32)
        table[have] = perm[:at]
        store[rows.long()] = table
        free = torch.zeros(blocks, dtype=torch.int32)
        free[:blocks - at] = perm[at:]
        dev = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
        s.update(store_t=store.cuda(), rows=rows.cuda(), starts=dev(starts), new_t=dev(new), total=sum(new), free=free.cuda(),
                 state=dev([0, blocks - at, 0, 0]), ends=dev([a + n for a, n in zip(starts, new)]), width=width)
        return s
    dt = _T[case["dtype"]]
    hq, hkv, dim, bs = case["hq"], case["hkv"], case["dim"], case["block"]
    if case["kind"] == "write":
        t = case["tokens"]
        blocks = -(-t // bs) + 9
        # one projection's output, split by columns: strided rows, as a fused q|k|v product gives
        qkv = torch.empty(t, (hq + 2 * hkv) * dim, device="cuda", dtype=dt).normal_(0, 1, generator=g)
        slots = torch.randperm(blocks * bs, generator=h)[:t]
        if case["pad"]:
            slots[t - case["pad"]:] = -1
        pos = torch.randint(0, 32768, (t,), generator=h).double().cuda()
        ang = pos[:, None] * (1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))[None, :]
        ang = torch.cat([ang, ang], dim=1)
        s.update(q=qkv[:, :hq * dim].view(t, hq, dim), k=qkv[:, hq * dim:(hq + hkv) * dim].view(t, hkv, dim), v=qkv[:, (hq + hkv) * dim:].view(t, hkv, dim),
                 cos=ang.cos().to(dt), sin=ang.sin().to(dt), slots=slots.cuda(),
                 codes=torch.randint(0, 256, (2, blocks, hkv, 2, bs, dim // 2), generator=g, device="cuda", dtype=torch.uint8),
                 params=torch.ones(2, blocks, hkv, 2, bs, 2, device="cuda", dtype=dt), layer=1)
        return s
    if case["kind"] == "decode":
        lens = _lengths(case, seed)
        tokens, cu = case["batch"], None
    else:
        new, lens = _chunks(case, seed)
        tokens = sum(new)
        cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        s.update(cu=cu, most=max(new))
    table, blocks = _tables(lens, bs, 11, h)
    codes, params = _pool(1, blocks, case, g)
    q = torch.empty(tokens, hq, dim, device="cuda", dtype=dt).normal_(0, 1, generator=g)
    s.update(q=q, codes=codes, params=params, table=table, lens_t=torch.tensor(lens, dtype=torch.int32).cuda(), layer=0)
    return s


# --------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------
def _quantize(x):
    """Codes (two a byte) and (step, mid) of rows ``x [..., D]``."""
    f = x.float()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    mid = (0.5 * lo + 0.5 * hi).to(x.dtype)
    m = mid.float()
    step = (torch.maximum(hi - m, m - lo) / 7.5).to(x.dtype)
    st = step.float()
    code = torch.where(st > 0, ((f - m) / st).floor() + 8, 8.0).clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([step, mid], -1)


def _values(codes, params):
    """The float32 values that codes ``[..., D / 2]`` and params ``[..., 2]`` stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.float()
    return p[..., 1:2] + p[..., 0:1] * (c - 7.5)


def _rotate(x, cos, sin):
    """x cos + rotate_half(x) sin, each product and the sum rounded to x's type: the rotary embedding's definition here."""
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    a = (x.float() * cos[:, None].float()).to(x.dtype)
    b = (turned.float() * sin[:, None].float()).to(x.dtype)
    return (a.float() + b.float()).to(x.dtype)


def _plain_write(s):
    q, k, v = s["q"], s["k"], s["v"]
    if s["rope"]:
        q, k = _rotate(q, s["cos"], s["sin"]), _rotate(k, s["cos"], s["sin"])
    codes, params = _quantize(torch.stack([k, v], 2))  # [T, Hkv, 2, .]
    live = s["slots"] >= 0
    at = s["slots"][live]
    blk, off = at // s["block"], at % s["block"]
    s["codes"][s["layer"]][blk, :, :, off] = codes[live]
    s["params"][s["layer"]][blk, :, :, off] = params[live]
    safe = s["slots"].clamp(min=0)
    blk, off = safe // s["block"], safe % s["block"]
    back = _values(s["codes"][s["layer"]][blk, :, :, off], s["params"][s["layer"]][blk, :, :, off])
    back = torch.where(live[:, None, None, None], back, 0.0).to(k.dtype)
    out = [back[:, :, 0], back[:, :, 1]]
    if s["rope"]:
        out += [q] + ([k] if s["keep_key"] else [])
    return out


def _plain_context(s):
    """The batch's keys and values [B, Hkv, W * BS, D] in float32, rows past a sequence's length zero."""
    t = s["table"].long()
    x = _values(s["codes"][s["layer"]][t], s["params"][s["layer"]][t])  # [B, W, Hkv, 2, BS, D]
    b, w, hkv, _, bs, d = x.shape
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, b, hkv, w * bs, d)
    have = torch.arange(w * bs, device=x.device)[None, :] < s["lens_t"][:, None]
    x = torch.where(have[None, :, None, :, None], x, 0.0)
    return x[0], x[1], have


def _plain_attend(q, k, v, mask):
    """softmax(q k^T / sqrt(D)) v over the last axes, rows with nothing to attend to zero."""
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = torch.where(mask, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _plain_decode(s):
    k, v, have = _plain_context(s)
    b, hkv, n, d = k.shape
    q = s["q"].float().view(b, hkv, s["hq"] // hkv, d)
    return _plain_attend(q, k, v, have[:, None, None, :]).reshape(b, s["hq"], d).to(s["q"].dtype)


def _plain_prefill(s):
    k, v, _ = _plain_context(s)
    b, hkv, n, d = k.shape
    cu = s["cu"].long()
    new = cu[1:] - cu[:-1]
    group = s["hq"] // hkv
    j = torch.arange(s["most"], device=k.device)
    live = j[None, :] < new[:, None]  # [B, most]
    rows = torch.where(live, cu[:-1, None] + j[None, :], 0)
    q = s["q"].float()[rows].view(b, s["most"], hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * s["most"], d)
    last = s["lens_t"].long()[:, None] - new[:, None] + j[None, :]  # the last position each row attends to
    mask = (torch.arange(n, device=k.device)[None, None, :] <= last[:, :, None]) & live[:, :, None]
    mask = mask[:, None, None].expand(b, 1, group, s["most"], n).reshape(b, 1, group * s["most"], n)
    o = _plain_attend(q, k, v, mask).view(b, hkv, group, s["most"], d).permute(0, 3, 1, 2, 4).reshape(b, s["most"], s["hq"], d)
    return o[live].to(s["q"].dtype)


def _plain_tables(s):
    bs, width = s["block"], s["width"]
    store, rows, starts, new = s["store_t"], s["rows"].long(), s["starts"].long(), s["new_t"].long()
    free, state = s["free"], s["state"]
    size = free.shape[0]
    held, ends = (starts + bs - 1) // bs, (starts + new + bs - 1) // bs
    grown = ends - held
    before = grown.cumsum(0) - grown
    head, count = state[0].long(), state[1].long()
    col = torch.arange(width, device=store.device)[None, :]
    fresh = (col >= held[:, None]) & (col < ends[:, None])
    take = free[(head + before[:, None] + col - held[:, None]).remainder(size)]
    table = torch.where(fresh, take, torch.where(col < held[:, None], store[rows], 0))
    store[rows] = torch.where(fresh, take, store[rows])
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    i = torch.arange(s["total"], device=store.device)
    b = torch.searchsorted(cu, i, right=True) - 1
    pos = starts[b] + i - cu[b]
    slots = table[b, pos // bs].long() * bs + pos % bs
    got = grown.sum()
    head, count = (head + got).remainder(size), count - got
    out = [cu.to(torch.int32), (starts + new).to(torch.int32), slots, pos, table]
    # give back the blocks past what the requests keep (here: what they held before)
    keep = (s["starts"].long() + bs - 1) // bs
    back = (col >= keep[:, None]) & (col < ends[:, None])
    many = ends - keep
    place = (head + count + (many.cumsum(0) - many)[:, None] + col - keep[:, None]).remainder(size)
    free[place[back]] = store[rows][back]
    store[rows] = torch.where(back, 0, store[rows])
    state[0], state[1] = head, count + many.sum()
    return out + [store, free, state]


# --------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"tables": _plain_tables, "write": _plain_write, "decode": _plain_decode, "prefill": _plain_prefill}[s["kind"]](s)
    from pagedserve_b200 import ops
    if s["kind"] == "tables":
        out = ops.extend_step(s["store_t"], s["rows"], s["starts"], s["new_t"], s["free"], s["state"], s["total"], s["block"], out_width=s["width"])
        ops.trim_tables(s["store_t"], s["rows"], s["ends"], s["starts"], s["free"], s["state"], s["block"])
        return list(out) + [s["store_t"], s["free"], s["state"]]
    if s["kind"] == "write":
        if s["rope"]:
            q, k = ops.rope_reshape_and_cache_int4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["codes"], s["params"], s["slots"], s["layer"],
                                                   key_out=None if s["keep_key"] else False)
        else:
            ops.reshape_and_cache_int4(s["k"], s["v"], s["codes"], s["params"], s["slots"], s["layer"])
        out = list(ops.gather_cache_int4(s["codes"], s["params"], s["slots"], s["layer"]))
        if s["rope"]:
            out += [q] + ([k] if s["keep_key"] else [])
        return out
    if s["kind"] == "decode":
        return ops.paged_decode_int4(s["q"], s["codes"], s["params"], s["table"], s["lens_t"], s["layer"])
    return ops.paged_prefill_int4(s["q"], s["codes"], s["params"], s["table"], s["lens_t"], s["cu"], s["most"], s["layer"])


# --------------------------------------------------------------------------------------------------------------
# 64 bits
# --------------------------------------------------------------------------------------------------------------
def _exact_rows(s, blocks, n):
    """Keys and values [Hkv, n, D] of one sequence in float64, from its block ids."""
    lay, d = s["layer"], s["dim"]
    pos = torch.arange(n, device=blocks.device)
    blk, off = blocks[pos // s["block"]].long(), pos % s["block"]
    c = s["codes"][lay, blk, :, :, off]  # [n, Hkv, 2, D / 2]
    v = torch.empty(*c.shape[:-1], d, dtype=torch.float64, device=c.device)
    v[..., 0::2] = (c % 16).double() - 7.5
    v[..., 1::2] = (c // 16).double() - 7.5
    p = s["params"][lay, blk, :, :, off].double()
    v = v * p[..., :1] + p[..., 1:]
    return v[:, :, 0].transpose(0, 1), v[:, :, 1].transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return None
    if case["kind"] == "write":
        dt = s["k"].dtype
        cos, sin = s["cos"].double()[:, None], s["sin"].double()[:, None]
        half = case["dim"] // 2
        turn = lambda x: torch.cat([-x[..., half:], x[..., :half]], -1)
        k, out = s["k"], []
        if case["rope"]:
            full = lambda x: x.double() * cos + turn(x.double()) * sin
            out = [full(s["q"])] + ([full(k)] if case["keep_key"] else [])
            k = ((k.double() * cos).to(dt).double() + (turn(k.double()) * sin).to(dt).double()).to(dt)  # what is stored is the rounded key
        live = (s["slots"] >= 0)[:, None, None]
        for i, x in enumerate((k, s["v"])):
            lo, hi = x.double().min(-1, keepdim=True)[0], x.double().max(-1, keepdim=True)[0]
            mid = ((lo + hi) / 2).float().to(dt)
            dev = torch.maximum(hi.float() - mid.float(), mid.float() - lo.float())
            step = (dev.double() / 7.5).float().to(dt)
            # which code is a decision: its two float32 roundings belong to the definition
            ratio = ((x.float() - mid.float()).double() / torch.where(step == 0, 1, step).double()).float()
            code = torch.where(step == 0, 8.0, (ratio.floor() + 8).clamp(0, 15)).double()
            val = mid.double() + step.double() * (code - 7.5)
            out.insert(i, torch.where(live, val, 0.0))
        return out
    group = case["hq"] // case["hkv"]
    lens = s["lens_t"].tolist()
    cu = s["cu"].tolist() if case["kind"] == "prefill" else list(range(case["batch"] + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        rows = cu[b + 1] - cu[b]
        if n == 0 or rows == 0:
            continue
        k, v = _exact_rows(s, s["table"][b], n)
        last = n - rows + torch.arange(rows, device="cuda")
        hide = torch.arange(n, device="cuda")[None, :] > last[:, None]
        for h in range(case["hkv"]):
            for j in range(group):
                a = s["q"][cu[b]:cu[b + 1], h * group + j].double() @ k[h].T / case["dim"] ** 0.5
                out[cu[b]:cu[b + 1], h * group + j] = torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v[h]
    return out
