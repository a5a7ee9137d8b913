"""What is measured of the operators that continue one prompt in several ways.

Three kinds of case, one pass each:

* ``pages``   continuations that start from a prompt's pages and end again: ``ops.fork_tables`` lets each child's row
              of the table store share its parent's whole blocks and gives it a block of its own for the unfinished
              one, ``ops.copy_blocks`` copies those blocks' keys and values in every layer, ``ops.release_tables``
              gives the children's pages back (a block when its last holder lets go of it);
* ``shared``  ``ops.paged_decode_shared``: one query token per sequence, the sequences of a group sharing their first
              pages, which are read and multiplied once for the whole group;
* ``verify``  ``ops.verify_tokens``: drafted tokens against the target's probabilities with given random numbers, the
              accepted ones and the token behind them; without drafts, sampling at a temperature.

The rule of ``verify``: row r of the logits, at temperature t, stands for p = softmax(logits[r] / t) (t = 0: all of it
on the first maximum).  The draft d behind row r, drawn from q (given as ``draft_probs[r]``; none: all of q on d), is
taken if u0[r] q(d) < p(d).  At the first row whose draft is not taken the new token is drawn from max(p - q, 0) (from p
where that is nothing), at a sequence's last row, or one with a draft below 0, from p: the first token whose cumulative
weight is above u1[r] times the weights' sum.
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
        # one prompt, a handful of candidates: latency
        dict(name="pages 4 of 1", kind="pages", parents=1, each=4, longest=777, siblings=0, store=64, layers=24, hkv=2, dim=64, block=16, dtype="bf16"),
        # every running prompt sampled several times, other continuations of the same prompts already there
        dict(name="pages 64 of 16", kind="pages", parents=16, each=4, longest=2000, siblings=1, store=512, layers=24, hkv=2, dim=64, block=16, dtype="bf16"),
        # a long shared prompt taken up by a full batch, wide heads, larger blocks
        dict(name="pages 255 of 3 f16", kind="pages", parents=3, each=85, longest=8000, siblings=2, store=1024, layers=2, hkv=8, dim=128, block=32, dtype="f16"),
        # a few samples of a short prompt: latency
        dict(name="shared 8 on 1k", kind="shared", groups=1, each=8, prefix=1000, own=64, empty=0, hq=14, hkv=2, dim=64, block=16, dtype="bf16"),
        # a prompt's 64 samples half way through their answers
        dict(name="shared 64 on 4k", kind="shared", groups=1, each=64, prefix=4096, own=700, empty=1, hq=14, hkv=2, dim=64, block=16, dtype="bf16"),
        # the served batch behind one system prompt, each with a conversation of its own
        dict(name="shared 256 on 2k", kind="shared", groups=1, each=256, prefix=2048, own=2000, empty=2, hq=14, hkv=2, dim=64, block=16, dtype="bf16"),
        # several prompts, each sampled eight times, in half precision; ragged prefixes that end inside a block
        dict(name="shared 32 x 8 on 1.5k f16", kind="shared", groups=32, each=8, prefix=1500, own=300, empty=0, hq=14, hkv=2, dim=64, block=16, dtype="f16"),
        # a long document and many questions, wide heads, groups of four, larger blocks
        dict(name="shared 96 on 30k d128", kind="shared", groups=1, each=96, prefix=30011, own=257, empty=0, hq=32, hkv=8, dim=128, block=32, dtype="bf16"),
        # one user, four tokens looked up in the prompt as drafts: latency
        dict(name="verify 1 x 4", kind="verify", batch=1, drafts=4, ragged=False, probs="", vocab=151936, dtype="bf16", greedy=0.0),
        # a served batch with a draft model, its probabilities kept in 32 bits, some of the users greedy
        dict(name="verify 32 x 5 probs", kind="verify", batch=32, drafts=5, ragged=True, probs="f32", vocab=151936, dtype="bf16", greedy=0.2),
        # many requests, short drafts, an odd vocabulary, half precision
        dict(name="verify 120 x 3 probs f16", kind="verify", batch=120, drafts=3, ragged=False, probs="f16", vocab=32003, dtype="f16", greedy=0.0),
        # plain sampling of a decode step: no drafts
        dict(name="verify 256 x 0", kind="verify", batch=256, drafts=0, ragged=False, probs="", vocab=151936, dtype="bf16", greedy=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["pages", "shared", "shared", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    hq, hkv, dim = rng.choice([(14, 2, 64), (14, 2, 64), (8, 8, 64), (12, 2, 64), (16, 1, 64), (32, 8, 128), (28, 4, 128), (10, 5, 64)])
    block = rng.choice([16, 16, 32])
    if kind == "pages":
        children = _log(rng, 1, 255)
        parents = _log(rng, 1, min(children, 20))
        longest = _log(rng, 1, max(1, min(8000, 24000 // parents)))
        return dict(kind=kind, parents=parents, each=children // parents, longest=longest, siblings=rng.randrange(0, 3), store=1024,
                    layers=rng.choice([1, 2, 4]) if hkv * dim > 128 else rng.choice([4, 12, 24]), hkv=hkv, dim=dim, block=block, dtype=dtype)
    if kind == "shared":
        batch = _log(rng, 1, 256)
        groups = rng.choice([1, 1, 2, _log(rng, 1, min(batch, 32))])
        each = max(1, batch // groups)
        room = 256 * 2 * 64 * 3000 // (groups * each * hkv * dim)
        prefix = _log(rng, 1, max(2, min(30000, 256 * 14 * 64 * 8000 // (groups * each * hq * dim))))
        return dict(kind=kind, groups=groups, each=each, prefix=prefix, own=_log(rng, 1, max(2, min(2000, room))), empty=rng.randrange(0, 1 + min(2, batch - 1)),
                    hq=hq, hkv=hkv, dim=dim, block=block, dtype=dtype)
    batch = _log(rng, 1, 256)
    drafts = rng.choice([0, 1, 2, 3, 4, 5, 7, 8])
    vocab = rng.choice([151936, 32003, _log(rng, 1000, 130000)])
    drafts = min(drafts, max(0, 128 * 151936 // (batch * vocab) - 1))
    return dict(kind=kind, batch=batch, drafts=drafts, ragged=drafts > 0 and rng.random() < 0.5, probs=rng.choice(["", "f32", "bf16"]) if drafts else "",
                vocab=vocab, dtype=rng.choice([dtype, dtype, "f32"]) if batch * vocab < 128 * 151936 else dtype, greedy=rng.choice([0.0, 0.0, 0.3]))


def _prompts(case, seed):
    """The parents' lengths of a pages case."""
    r = random.Random(seed * 7 + 1)
    return [max(1, case["longest"] - r.randrange(0, 1 + case["longest"] // 3)) for _ in range(case["parents"])]


def _groups(case, seed):
    """(prefix lengths of the groups, lengths of the sequences) of a shared case."""
    r = random.Random(seed * 7 + 2)
    prefix = [max(1, case["prefix"] - (r.randrange(0, 1 + case["prefix"] // 4) if case["groups"] > 1 else r.randrange(0, 1 + case["prefix"] // 100))) for _ in range(case["groups"])]
    lens = [p + r.randint(1, case["own"]) for p in prefix for _ in range(case["each"])]
    idle = {(i * 97 + 1) % len(lens) for i in range(case["empty"])}
    return prefix, [0 if i in idle else n for i, n in enumerate(lens)]


def _drafts(case, seed):
    """Drafts of each sequence of a verify case: a case's own counts, in an order of the seed's."""
    r, own_r = random.Random(seed * 7 + 3), random.Random(case["batch"] * 1009 + case["drafts"])
    n = [own_r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["batch"])]
    r.shuffle(n)
    return n


def work(case):
    e = _SIZE[case["dtype"]]
    if case["kind"] == "pages":
        lens, bs = _prompts(case, 0), case["block"]
        full, part = sum(n // bs for n in lens), sum(1 for n in lens if n % bs)
        held = case["each"] * (full + part)
        # plan in; parents' entries and counts read and written; children's entries written, read and cleared; the
        # blocks copied, in and out
        return dict(bytes=4 * 6 * case["parents"] * case["each"] + 4 * 5 * full + 12 * held
                    + 2 * case["each"] * part * case["layers"] * 2 * case["hkv"] * bs * case["dim"] * e, flops=0)
    if case["kind"] == "shared":
        prefix, lens = _groups(case, 0)
        each = case["each"]
        rest = sum(max(0, n - prefix[i // each]) for i, n in enumerate(lens))
        row = 2 * case["hkv"] * case["dim"] * e
        return dict(bytes=(sum(prefix) + rest) * row + 2 * len(lens) * case["hq"] * case["dim"] * e + 4 * (sum(prefix) + rest) // case["block"],
                    flops=4 * case["hq"] * case["dim"] * sum(lens))
    # rows up to a first rejection, seven drafts in ten being taken, and the draft's probabilities there
    n, v = _drafts(case, 0), case["vocab"]
    rows = sum(sum(0.7 ** i for i in range(k + 1)) for k in n)
    turned = sum(1 - 0.7 ** k for k in n) if case["probs"] else 0
    return dict(bytes=int(rows * v * e + (turned * v * _SIZE[case["probs"]] if case["probs"] else 0)) + 24 * (sum(n) + len(n)), flops=int(4 * rows * v))


# --------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 13 + 5)
    h = torch.Generator()
    h.manual_seed(seed * 17 + 7)
    s = dict(case)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    if case["kind"] == "pages":
        lens, bs, each = _prompts(case, seed), case["block"], case["each"]
        width = -(-case["longest"] // bs) + 3
        need = [-(-n // bs) for n in lens]
        blocks = case["parents"] * (-(-case["longest"] // bs) + each + case["siblings"]) + 9
        perm = torch.randperm(blocks, generator=h).to(torch.int32)
        rows = torch.randperm(case["store"], generator=h).to(torch.int32)
        store = torch.zeros(case["store"], width, dtype=torch.int32)
        shares = torch.zeros(2, blocks, dtype=torch.int32)
        at, used = 0, case["parents"] * (1 + case["siblings"])
        for i, (n, k) in enumerate(zip(lens, need)):
            store[rows[i], :k] = perm[at:at + k]
            shares[0, perm[at:at + n // bs].long()] = case["siblings"]
            at += k
        for i in range(case["parents"] * case["siblings"]):  # continuations that are there already
            p = i % case["parents"]
            row = rows[case["parents"] + i]
            store[row, :lens[p] // bs] = store[rows[p], :lens[p] // bs]
            if lens[p] % bs:
                store[row, lens[p] // bs] = perm[at]
                at += 1
        free = torch.zeros(blocks, dtype=torch.int32)
        free[:blocks - at] = perm[at:]
        order = [p for p in range(case["parents"]) for _ in range(each)]
        random.Random(seed * 7 + 4).shuffle(order)
        shape = (case["layers"], blocks, case["hkv"], bs, case["dim"])
        pool = lambda: torch.empty(shape, device="cuda", dtype=_T[case["dtype"]]).normal_(0, 1, generator=g)
        s.update(store_t=store.cuda(), shares=shares.cuda(), free=free.cuda(), state=i32([0, blocks - at, 0, 0]),
                 parents_t=rows[torch.tensor(order)].cuda(), children_t=rows[used:used + len(order)].cuda(), lens_t=i32([lens[p] for p in order]),
                 none_t=i32([0] * len(order)), k=pool(), v=pool())
        return s
    if case["kind"] == "shared":
        prefix, lens = _groups(case, seed)
        bs, dt = case["block"], _T[case["dtype"]]
        whole = [p // bs for p in prefix]
        alone = [max(0, -(-n // bs) - whole[i // case["each"]]) for i, n in enumerate(lens)]
        blocks = sum(whole) + sum(alone) + 11
        perm = torch.randperm(blocks, generator=h).to(torch.int32)
        table = torch.zeros(len(lens), max(1, -(-max(lens) // bs)), dtype=torch.int32)
        at, first = sum(whole), 0
        starts = []
        for w in whole:
            starts.append(first)
            first += w
        for i, n in enumerate(lens):
            w = whole[i // case["each"]]
            if n:
                a = starts[i // case["each"]]
                table[i, :w] = perm[a:a + w]
                table[i, w:w + alone[i]] = perm[at:at + alone[i]]
            at += alone[i]
        shape = (2, blocks, case["hkv"], bs, case["dim"])
        k = torch.empty(shape, device="cuda", dtype=dt).normal_(0, 1, generator=g)
        v = torch.empty(shape, device="cuda", dtype=dt).normal_(0, 1, generator=g)
        k[..., 5] += 4.0  # a channel that stands out, as biased key projections give
        table = table.cuda()
        # a prefix that ends inside a block: its last rows are each sequence's own copy, the same in all of them
        for i, n in enumerate(lens):
            j = i // case["each"]
            lead = next((m for m in range(j * case["each"], (j + 1) * case["each"]) if lens[m]), i)
            if n and i != lead and prefix[j] % bs:
                a, b = int(table[lead, whole[j]]), int(table[i, whole[j]])
                for pool in (k, v):
                    pool[:, b, :, :prefix[j] % bs] = pool[:, a, :, :prefix[j] % bs]
        q = torch.empty(len(lens), case["hq"], case["dim"], device="cuda", dtype=dt).normal_(0, 1, generator=g)
        s.update(q=q, k=k, v=v, table=table, lens_t=i32(lens), cu=i32(list(range(0, len(lens) + 1, case["each"]))), prefix_t=i32(prefix), layer=1)
        return s
    n, vocab, dt = _drafts(case, seed), case["vocab"], _T[case["dtype"]]
    total = sum(n) + len(n)
    cu = [0]
    for k in n:
        cu.append(cu[-1] + k + 1)
    r = random.Random(seed * 7 + 5)
    heat = [0.0 if r.random() < case["greedy"] else r.uniform(0.6, 1.2) for _ in n]
    # spread-out logits and one token in each row that stands out
    logits = torch.empty(total, vocab, device="cuda").normal_(0, 2, generator=g)
    peak = torch.randint(0, vocab, (total, 1), generator=h).cuda()
    logits.scatter_(1, peak, math.log(vocab) + 2 + 1 + torch.empty(total, 1, device="cuda").normal_(0, 1, generator=g))
    logits = logits.to(dt)
    seq = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n) + 1).cuda()
    t_row = torch.tensor(heat, device="cuda")[seq][:, None]
    tokens = torch.randint(0, vocab, (total,), generator=h).cuda()
    probs = None
    if case["probs"]:
        probs = torch.empty(total, vocab, device="cuda", dtype=_T[case["probs"]])
    drawn = peak[:, 0].clone()
    for a in range(0, total, 64) if case["probs"] else ():  # what a smaller model makes of the same rows
        z = logits[a:a + 64].float()
        z += torch.empty_like(z).normal_(0, 0.7, generator=g)
        q = torch.softmax(z / torch.where(t_row[a:a + 64] > 0, t_row[a:a + 64], 0.3), -1).to(probs.dtype)
        probs[a:a + 64] = q
        drawn[a:a + 64] = (q.float() / torch.empty_like(z).exponential_(generator=g)).argmax(-1)
    tokens[1:] = drawn[:-1]  # the draft behind each row (a sequence's first token is none: it is not looked at)
    s.update(logits=logits, tokens=tokens, cu=i32(cu), uniforms=torch.rand(total, 2, device="cuda", generator=g), heat=torch.tensor(heat, dtype=torch.float32).cuda(), probs_t=probs)
    return s


# --------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------
def _plain_pages(s):
    bs, store, free, state, shares = s["block"], s["store_t"], s["free"], s["state"], s["shares"]
    size, width = free.shape[0], store.shape[1]
    parents, children, lens = s["parents_t"].long(), s["children_t"].long(), s["lens_t"].long()
    col = torch.arange(width, device=store.device)[None, :]
    # fork: whole blocks are shared, an unfinished one gets a block of its own from the head of the free ring
    full, part = lens // bs, lens % bs > 0
    head, count = state[0].long(), state[1].long()
    before = part.long().cumsum(0) - part.long()
    fresh = free[(head + before).remainder(size)]
    held = store[parents]
    table = torch.where(col < full[:, None], held, 0)
    unfinished = (col == full[:, None]) & part[:, None]
    table = torch.where(unfinished, fresh[:, None], table)
    store[children] = table
    shares[0].index_put_((held[col < full[:, None]].long(),), torch.ones((), dtype=torch.int32, device=store.device), accumulate=True)
    src = torch.where(part, held.gather(1, full.clamp(max=width - 1)[:, None])[:, 0], -1)
    dst = torch.where(part, fresh, -1)
    head, count = (head + part.sum()).remainder(size), count - part.sum()
    # copy
    for pool in (s["k"], s["v"]):
        pool[:, dst[part].long()] = pool[:, src[part].long()]
    # release, entry by entry: a block goes to the tail of the ring with the last of its holders
    back = col < ((lens + bs - 1) // bs)[:, None]
    ids = table[back].long()
    times = torch.zeros(size, dtype=torch.int64, device=store.device).index_put_((ids,), torch.ones((), dtype=torch.int64, device=store.device), accumulate=True)
    order = torch.arange(ids.shape[0], device=store.device)
    last = torch.full((size,), -1, dtype=torch.int64, device=store.device).scatter_reduce_(0, ids, order, "amax")
    gone = (times > shares[0]) & (times > 0)
    freed = ids[gone[ids] & (last[ids] == order)]
    free[(head + count + torch.arange(freed.shape[0], device=store.device)).remainder(size)] = freed.to(torch.int32)
    shares[0] = torch.where(gone, 0, shares[0] - times).to(torch.int32)
    store[children] = 0
    state[0], state[1] = head, count + freed.shape[0]
    return [src.to(torch.int32), dst.to(torch.int32), store, shares, free, state, s["k"], s["v"]]


def _plain_shared(s):
    q, table, lens = s["q"], s["table"].long(), s["lens_t"].long()
    k, v = s["k"][s["layer"]], s["v"][s["layer"]]
    b, hq, d = q.shape
    hkv, bs = k.shape[1], k.shape[2]
    group, cu, prefix = hq // hkv, s["cu"].long(), s["prefix_t"].long()
    count = torch.arange(table.shape[1] * bs, device=q.device)
    seq = torch.arange(b, device=q.device)
    j = torch.searchsorted(cu, seq, right=True) - 1
    # the pages of a prefix, from the table of the group's longest sequence, once for the group
    member = torch.where(j[None, :] == torch.arange(cu.shape[0] - 1, device=q.device)[:, None], lens[None, :], -1)
    lead = member.argmax(1)
    most = torch.minimum(prefix, member.amax(1))
    out = torch.empty(b, hq, d, dtype=q.dtype, device=q.device)
    each = s["each"]  # sequences of a group: every group has as many
    span = 512 if b * hq * table.shape[1] * bs < 1 << 28 else 64  # sequences at a time, for the memory they take
    gp = s["groups"]
    width = -(-s["prefix"] // bs)
    pos = count[:width * bs]
    see = pos[None, :] < most[:, None]
    rows = lambda pool, t: pool[t].permute(0, 2, 1, 3, 4).reshape(t.shape[0], hkv, -1, d).float()
    zero = lambda x, keep: torch.where(keep[:, None, :, None], x, 0.0)
    kp, vp = zero(rows(k, table[lead, :width]), see), zero(rows(v, table[lead, :width]), see)
    qg = q.float().view(gp, each, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(gp, hkv, each * group, d)
    sp = torch.matmul(qg, kp.transpose(-1, -2)) / math.sqrt(d)
    mask = (see[:, None, :] & (pos[None, None, :] < lens.view(gp, each)[:, :, None])).repeat_interleave(group, 1)
    sp = torch.where(mask[:, None], sp, -math.inf)
    back = lambda x: x.view(gp, hkv, each, group, -1).permute(0, 2, 1, 3, 4).reshape(b, hkv, group, -1)
    top = sp.amax(-1, keepdim=True)
    e = torch.exp(sp - torch.where(top == -math.inf, 0.0, top))
    top_p, sum_p, o_p = back(top), back(e.sum(-1, keepdim=True)), back(torch.matmul(e, vp))
    # what is each sequence's own
    for a in range(0, b, span):
        n, f = lens[a:a + span], most[j[a:a + span]]
        at = f[:, None] // bs + torch.arange(-(-s["own"] // bs) + 1, device=q.device)[None, :]
        t = torch.where(at < table.shape[1], table[a:a + span].gather(1, at.clamp(max=table.shape[1] - 1)), 0)
        pos = (at[:, :, None] * bs + torch.arange(bs, device=q.device)).reshape(t.shape[0], -1)
        see = (pos >= f[:, None]) & (pos < n[:, None])
        ks, vs = zero(rows(k, t), see), zero(rows(v, t), see)
        ss = torch.matmul(q[a:a + span].float().view(-1, hkv, group, d), ks.transpose(-1, -2)) / math.sqrt(d)
        ss = torch.where(see[:, None, None, :], ss, -math.inf)
        top = torch.maximum(ss.amax(-1, keepdim=True), top_p[a:a + span])
        top = torch.where(top == -math.inf, 0.0, top)
        e, w = torch.exp(ss - top), torch.exp(top_p[a:a + span] - top)
        total = e.sum(-1, keepdim=True) + w * sum_p[a:a + span]
        o = torch.matmul(e, vs) + w * o_p[a:a + span]
        out[a:a + span] = (o / torch.where(total == 0, 1.0, total)).view(-1, hq, d).to(q.dtype)
    return out


def _plain_verify(s):
    # in 64 bits: which token a random number falls on is decided next to a border
    logits, cu, u = s["logits"], s["cu"].long(), s["uniforms"].double()
    total, vocab = logits.shape
    b = cu.shape[0] - 1
    rows = torch.arange(total, device=logits.device)
    seq = torch.searchsorted(cu, rows, right=True) - 1
    t = s["heat"].double()[seq]
    draft = torch.cat([s["tokens"][1:], s["tokens"].new_full((1,), -1)])
    draft = torch.where(rows + 1 < cu[seq + 1], draft, -1)
    arg = torch.empty_like(rows)  # the first maximum of each row
    for a in range(0, total, 256):
        x = logits[a:a + 256]
        arg[a:a + 256] = torch.where(x == x.amax(-1, keepdim=True), torch.arange(vocab, device=x.device), vocab).amin(-1)
    taken = torch.zeros(total, dtype=torch.bool, device=logits.device)

    def probabilities(r):
        x = logits[r].double() / torch.where(t[r] > 0, t[r], 1.0)[:, None]
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        return torch.where((t[r] > 0)[:, None], p, (torch.arange(vocab, device=p.device)[None, :] == arg[r][:, None]).double())

    for a in range(0, total, 256):
        r = rows[a:a + 256]
        d = draft[r].clamp(min=0)[:, None]
        q = s["probs_t"][r].gather(1, d)[:, 0].double() if s["probs_t"] is not None else 1.0
        taken[r] = (u[r, 0] * q < probabilities(r).gather(1, d)[:, 0]) & (draft[r] >= 0)
    stops = torch.where(taken, total, rows)  # a sequence's first row whose draft is not taken
    stop = torch.full((b,), total, dtype=torch.int64, device=logits.device).scatter_reduce_(0, seq, stops, "amin")
    new = torch.empty(b, dtype=torch.int64, device=logits.device)
    for a in range(0, b, 256):
        r = stop[a:a + 256]
        p = probabilities(r)
        d = draft[r]
        if s["probs_t"] is not None:
            q = s["probs_t"][r].double()
        else:
            q = (torch.arange(vocab, device=p.device)[None, :] == d[:, None]).double()
        w = torch.where((d >= 0)[:, None], (p - q).clamp(min=0), p)
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
        c = w.cumsum(-1)
        at = (c <= u[r, 1:2] * c[:, -1:]).sum(-1)
        last = torch.where(w > 0, torch.arange(vocab, device=p.device), -1).amax(-1)
        new[a:a + 256] = torch.minimum(at, last)
    out = torch.where(rows < stop[seq], draft, -1)
    out[stop] = new
    return [out, (stop - cu[:-1] + 1).to(torch.int32)]


# --------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"pages": _plain_pages, "shared": _plain_shared, "verify": _plain_verify}[s["kind"]](s)
    from pagedserve_b200 import ops
    if s["kind"] == "pages":
        src, dst = ops.fork_tables(s["store_t"], s["parents_t"], s["children_t"], s["lens_t"], s["shares"], s["free"], s["state"], s["block"])
        ops.copy_blocks((s["k"], s["v"]), src, dst)
        ops.release_tables(s["store_t"], s["children_t"], s["lens_t"], s["none_t"], s["shares"], s["free"], s["state"], s["block"])
        return [src, dst, s["store_t"], s["shares"], s["free"], s["state"], s["k"], s["v"]]
    if s["kind"] == "shared":
        return ops.paged_decode_shared(s["q"], s["k"], s["v"], s["table"], s["lens_t"], s["cu"], s["prefix_t"], s["layer"])
    return list(ops.verify_tokens(s["logits"], s["tokens"], s["cu"], s["uniforms"], s["heat"], draft_probs=s["probs_t"]))


# --------------------------------------------------------------------------------------------------------------
# 64 bits
# --------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers and copies
    s = prepare(case, seed)
    if case["kind"] == "shared":
        lay, bs, group = s["layer"], case["block"], case["hq"] // case["hkv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(s["lens_t"].tolist()):
            if n == 0:
                continue
            blk = s["table"][i, :-(-n // bs)].long()
            k, v = (x[lay, blk].transpose(0, 1).reshape(case["hkv"], -1, case["dim"])[:, :n].double() for x in (s["k"], s["v"]))
            for h in range(case["hkv"]):
                a = s["q"][i, h * group:(h + 1) * group].double() @ k[h].T / case["dim"] ** 0.5
                out[i, h * group:(h + 1) * group] = torch.softmax(a, -1) @ v[h]
        return out
    cu, draft, u, heat = s["cu"].tolist(), s["tokens"].tolist(), s["uniforms"].double().tolist(), s["heat"].double().tolist()
    out, counts = torch.full((cu[-1],), -1, dtype=torch.int64), []
    for b in range(case["batch"]):
        for r in range(cu[b], cu[b + 1]):
            x = s["logits"][r].double()
            if heat[b] > 0:
                p = torch.softmax(x / heat[b], 0)
            else:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
            w = p
            if r + 1 < cu[b + 1]:
                d = draft[r + 1]
                if s["probs_t"] is None:
                    q = torch.zeros_like(p)
                    q[d] = 1.0
                else:
                    q = s["probs_t"][r].double()
                if u[r][0] * float(q[d]) < float(p[d]):
                    out[r] = d
                    continue
                w = torch.relu(p - q)
                if float(w.sum()) == 0:
                    w = p
            c = torch.cumsum(w, 0)
            out[r] = int(torch.searchsorted(c, u[r][1] * c[-1:], right=True).clamp(max=int(w.nonzero()[-1])))
            counts.append(r - cu[b] + 1)
            break
    return [out.cuda(), torch.tensor(counts, dtype=torch.int32).cuda()]
