"""The 4-bit pool's and the block tables' entry points called in the ways the
native fast call does not take (strides, types of arguments, subclasses, other
streams): the same results as the ordinary call, or the error's wording."""

from __future__ import annotations

import pytest
import torch

from pagedserve_b200 import _native, ops
from tests import int4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


class _Sub(torch.Tensor):
    pass


def _strided(t):
    """Equal values, twice the stride along the last axis."""
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def _case(seed=5, hq=14, hkv=2, d=64, bs=16):
    gen = torch.Generator().manual_seed(seed)
    lens = [70, 1, 200]
    table, blocks = ref.shuffled_tables(gen, lens, bs)
    codes, params = ref.make_pool(gen, 2, blocks, hkv, bs, d, torch.bfloat16)
    rnd = lambda *s: torch.randn(*s, generator=gen).bfloat16().cuda()
    return dict(codes=codes.cuda(), params=params.cuda(), table=table.cuda(),
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), q=rnd(3, hq, d), k=rnd(3, hkv, d),
                v=rnd(3, hkv, d), cos=rnd(3, d), sin=rnd(3, d),
                slots=torch.tensor([5, -1, 40], device="cuda"), cu=torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"))


def test_native_calls_are_loaded():
    assert _native.calls().__file__.startswith(_native.LIB_PATH.rsplit("/", 1)[0])


def test_attention_takes_other_layouts_and_arguments():
    c = _case()
    args = (c["codes"], c["params"], c["table"], c["lens"], 1)
    want = ops.paged_decode_int4(c["q"], *args, scale=1.0)
    assert torch.equal(ops.paged_decode_int4(c["q"], *args, scale=1), want)
    assert torch.equal(ops.paged_decode_int4(_strided(c["q"]), *args, scale=1.0), want)
    assert torch.equal(ops.paged_decode_int4(c["q"].as_subclass(_Sub), *args, scale=1.0), want)
    assert torch.equal(ops.paged_decode_int4(torch.nn.Parameter(c["q"]), *args, scale=1.0), want)
    assert torch.equal(ops.paged_decode_int4(c["q"], c["codes"], c["params"], _strided(c["table"]), _strided(c["lens"]), 1,
                                             scale=1.0), want)
    assert torch.equal(ops.paged_decode_int4(c["q"].unsqueeze(2), *args, scale=1.0), want.unsqueeze(2))
    swapped = c["q"].transpose(0, 1).contiguous().transpose(0, 1)  # dense, heads outermost
    assert torch.equal(ops.paged_decode_int4(swapped, *args, scale=1.0), want)
    out = torch.empty(3, 14, 128, dtype=torch.bfloat16, device="cuda")[..., :64]
    assert ops.paged_decode_int4(c["q"], *args, scale=1.0, out=out) is out and torch.equal(out, want)
    ws = torch.empty(ops.decode_int4_workspace_bytes(3, 14, 2, 64, 16, c["table"].shape[1] * 16, torch.bfloat16),
                     dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.paged_decode_int4(c["q"], *args, scale=1.0, workspace=ws), want)
    want = ops.paged_prefill_int4(c["q"], *args[:4], c["cu"], 1, 1, scale=1.0)
    for q, cu in ((_strided(c["q"]), c["cu"]), (c["q"], _strided(c["cu"])), (swapped, c["cu"])):
        assert torch.equal(ops.paged_prefill_int4(q, *args[:4], cu, 1, 1, scale=1), want)


def test_writes_take_other_layouts():
    c = _case()
    slots = c["slots"]

    def run(q, k, v, cos, sin, slots, **kw):
        codes, params = c["codes"].clone(), c["params"].clone()
        qo, ko = ops.rope_reshape_and_cache_int4(q, k, v, cos, sin, codes, params, slots, 1, **kw)
        return codes, params, qo, ko, *ops.gather_cache_int4(codes, params, slots, 1)

    want = run(c["q"], c["k"], c["v"], c["cos"], c["sin"], slots)
    wide = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda")
    sin = wide[:, :64].copy_(c["sin"])  # another row stride than cos
    for got in (run(c["q"], c["k"], c["v"], c["cos"].unsqueeze(1), c["sin"].unsqueeze(1), slots),
                run(c["q"], c["k"], c["v"], c["cos"], sin, slots),
                run(c["q"].as_subclass(_Sub), c["k"], c["v"], c["cos"], c["sin"], _strided(slots)),
                run(c["q"], c["k"], c["v"], c["cos"], c["sin"], slots, query_out=torch.empty_like(c["q"]),
                    key_out=torch.empty_like(c["k"]))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = run(c["q"], c["k"], c["v"], c["cos"], c["sin"], slots, key_out=False)
    assert none[3] is None and all(torch.equal(a, b) for i, (a, b) in enumerate(zip(none, want)) if i != 3)


def test_errors_keep_their_wording():
    c = _case()
    args = (c["codes"], c["params"], c["table"], c["lens"])
    with pytest.raises(ValueError, match="every tensor must be on cuda"):
        ops.paged_decode_int4(c["q"], c["codes"], c["params"], c["table"].cpu(), c["lens"], 0)
    with pytest.raises(ValueError, match="Invalid layer"):
        ops.paged_decode_int4(c["q"], *args, 2)
    with pytest.raises(ValueError, match="Query dtype"):
        ops.paged_decode_int4(c["q"].half(), *args, 0)
    with pytest.raises(ValueError, match="max_context"):
        ops.paged_decode_int4(c["q"], *args, 0, max_context=10 ** 6)
    with pytest.raises(ValueError, match="max_seqlen"):
        ops.paged_prefill_int4(c["q"], *args, c["cu"], 10 ** 6, 0)
    with pytest.raises(_native.NativeError, match="paged_decode_int4"):
        ops.paged_decode_int4(c["q"], *args, 0, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="slot_mapping must be int64"):
        ops.reshape_and_cache_int4(c["k"], c["v"], c["codes"], c["params"], c["slots"].int(), 0)
    store = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    free, state = ops.free_list(16, "cuda")
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="free_state"):
        ops.extend_step(store, rows, rows, rows, free, state[:3], 0, 16)
    with pytest.raises(ValueError, match="block_size"):
        ops.trim_tables(store, rows, rows, rows, free, state, 0)


def test_tables_on_another_stream_and_strided_plans():
    def run(stream, view):
        store = torch.zeros(6, 12, dtype=torch.int32, device="cuda")
        free, state = ops.free_list(40, "cuda")
        plan = [view(torch.tensor(x, dtype=torch.int32, device="cuda")) for x in ([4, -1, 0], [0, 0, 0], [33, 2, 16], [1, 0, 16])]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out = ops.extend_step(store, plan[0], plan[1], plan[2], free, state, 51, 16)
            ops.trim_tables(store, plan[0], plan[2], plan[3], free, state, 16)
        torch.cuda.synchronize()
        return list(out) + [store, free, state]

    want = run(torch.cuda.current_stream(), lambda t: t)
    for got in (run(torch.cuda.Stream(), lambda t: t), run(torch.cuda.Stream(), _strided)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def _calls_of(c):
    """One call of each entry point, by name."""
    store = torch.zeros(6, 12, dtype=torch.int32, device="cuda")
    free, state = ops.free_list(40, "cuda")
    rows, zero, one = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (2, 0, 1))
    pool = (c["codes"], c["params"])
    return {
        "write": lambda: ops.reshape_and_cache_int4(c["k"], c["v"], *pool, c["slots"], 1),
        "rope_write": lambda: ops.rope_reshape_and_cache_int4(c["q"], c["k"], c["v"], c["cos"], c["sin"], *pool, c["slots"], 1),
        "gather": lambda: ops.gather_cache_int4(*pool, c["slots"], 1),
        "decode": lambda: ops.paged_decode_int4(c["q"], *pool, c["table"], c["lens"], 1),
        "prefill": lambda: ops.paged_prefill_int4(c["q"], *pool, c["table"], c["lens"], c["cu"], 1, 1),
        "extend": lambda: ops.extend_step(store, rows, zero, zero, free, state, 0, 16),
        "trim": lambda: ops.trim_tables(store, rows, zero, zero, free, state, 16),
    }


@pytest.mark.parametrize("name", ["write", "rope_write", "gather", "decode", "prefill", "extend", "trim"])
def test_a_full_launch_queue_stops_no_other_thread(name):
    """A thread that waits for room in its stream's launch queue leaves the
    interpreter to the others: behind a kernel of about a second, more calls
    than the queue holds, and a second thread that looks at the clock."""
    import threading
    import time
    call = _calls_of(_case())[name]
    call()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    took = []

    def launches():
        begin = time.perf_counter()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(1_500_000_000)
            for _ in range(1500):
                call()
        took.append(time.perf_counter() - begin)

    worker = threading.Thread(target=launches)
    worker.start()
    last, gap = time.perf_counter(), 0.0
    while worker.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        last, gap = now, max(gap, now - last)
    worker.join()
    torch.cuda.synchronize()
    assert took[0] > 0.4  # the queue was full, most of that time
    assert gap < took[0] / 2
