"""Rotary positions, appending to a paged cache and attention over it on the GPU, against the definitions in 64 bits."""
import math
import os

import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def nothing_gave_up():
    yield
    from glq_b200 import ops
    ops.paged_check_status()


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _close(y, ref, bound, what=""):
    """Within the bound, and not a number exactly where the definition has none."""
    y = y.double().cpu()
    assert torch.equal(y.isnan(), ref.isnan()) and not y.isinf().any(), what
    err = ((y - ref).abs() - bound).nan_to_num(0.0)
    assert float(err.max()) <= 0, (what, float(err.max()), int(err.argmax()))


def _freq(dim, base=10000.0):
    return base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)


# ---- rotary -------------------------------------------------------------------------------------------------------
U = {BF: 2.0 ** -8, HF: 2.0 ** -11, F32: 2.0 ** -24}


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 20, 128, 128), (3, 5, 64, 32), (257, 3, 80, 40), (33, 2, 96, 24), (7, 1, 66, 30), (5000, 1, 8, 2), (2, 300, 256, 256)])
def test_rotary(dtype, interleaved, tokens, heads, dim, rot):
    from glq_b200 import ops
    g = _gen(tokens + dim)
    x = _randn(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(0, 1_000_000, (tokens,), generator=g, device="cuda")
    pos = pos if tokens % 2 else pos.to(torch.int32)
    y = ops.rotary(x, pos, ops.rotary_table(rot, interleaved=interleaved, scale=1.25))
    ref, mag = O.rotate(x, pos, _freq(rot), 1.25, interleaved)
    assert y.shape == x.shape and y.dtype == dtype
    _close(y, ref, mag + (ref.abs() + mag) * U[dtype])
    assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_far_positions_and_back():
    from glq_b200 import ops
    x = _randn(_gen(), 6, 4, 128, dtype=F32)
    table = ops.rotary_table(128, base=5e6)
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -7], device="cuda")
    y = ops.rotary(x, pos, table)
    # (a frequency in 64 bits is off by 2^-53 of itself: at 2^40 by 2^-13 turns; the reference takes the table's own turns)
    ref = x.double().cpu().clone()
    for i, t in enumerate(table.turns.cpu().tolist()):
        for r, p in enumerate(pos.cpu().tolist()):
            part = (t * p) % 2 ** 64
            a = 2 * math.pi * (part - 2 ** 64 if part >= 2 ** 63 else part) / 2 ** 64
            u, v = x[r, :, i].double().cpu(), x[r, :, i + 64].double().cpu()
            ref[r, :, i], ref[r, :, i + 64] = u * math.cos(a) - v * math.sin(a), v * math.cos(a) + u * math.sin(a)
    mag = (x.double().cpu()[..., :64].abs() + x.double().cpu()[..., 64:].abs()).repeat(1, 1, 2)
    _close(y, ref, mag * 2.0 ** -20)
    assert torch.equal(y[0], x[0])
    _close(ops.rotary(y, -pos, table), x.double().cpu(), mag * 2.0 ** -18)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("off,width", [(0, 512), (64, 640), (1, 513), (3, 700)])
def test_rotary_strides_alignment_and_in_place(dtype, off, width):
    from glq_b200 import ops
    g = _gen(off)
    buf = _randn(g, 50, width, dtype=dtype)
    x = torch.as_strided(buf.flatten()[off:], (49, 4, 96), (width, 128, 1))       # heads apart, rows of a wider matrix
    pos, table = torch.arange(49, device="cuda"), ops.rotary_table(64)
    want = ops.rotary(x.contiguous(), pos, table)
    assert torch.equal(ops.rotary(x, pos, table), want)
    out = torch.full_like(buf, 7.0)
    into = torch.as_strided(out.flatten()[off:], x.shape, x.stride())
    assert ops.rotary(x, pos, table, out=into) is into and torch.equal(into, want)
    into.fill_(7.0)
    assert bool((out == 7.0).all())                                               # nothing beside the rows was written
    assert torch.equal(ops.rotary(x, pos, table, out=x), want) and torch.equal(x, want)
    assert torch.equal(ops.rotary(x.transpose(1, 2).contiguous().transpose(1, 2), pos, table), ops.rotary(x, pos, table))


# ---- append -------------------------------------------------------------------------------------------------------
def _caches(g, pages, size, kv, dim, dtype, layout="rows"):
    """A pair of caches: rows (pages, size, kv, dim), or heads first within a page, or both in one tensor."""
    if layout == "rows":
        return _randn(g, pages, size, kv, dim, dtype=dtype), _randn(g, pages, size, kv, dim, dtype=dtype)
    if layout == "heads":
        return tuple(_randn(g, pages, kv, size, dim, dtype=dtype).transpose(1, 2) for _ in range(2))
    both = _randn(g, pages, 2, size, kv, dim + 8, dtype=dtype)
    return both[:, 0, ..., :dim], both[:, 1, ..., :dim]


@pytest.mark.parametrize("layout", ["rows", "heads", "both"])
@pytest.mark.parametrize("source", ["own", "fp32"])
@pytest.mark.parametrize("dtype,tokens,heads,kv,dim,size,rot", [(BF, 1, 16, 4, 128, 16, 128), (HF, 300, 6, 2, 64, 8, 32), (BF, 37, 5, 1, 72, 32, 36), (HF, 6000, 2, 2, 16, 64, 16)])
def test_append(layout, source, dtype, tokens, heads, kv, dim, size, rot):
    from glq_b200 import ops
    g, kind = _gen(tokens), dtype if source == "own" else F32
    pages = -(-tokens // size) + 5
    keys, values = _caches(g, pages, size, kv, dim, dtype, layout)
    before = keys.clone(), values.clone()
    merged = _randn(g, tokens, (heads + 2 * kv) * dim, dtype=kind)                 # a q/k/v projection's result
    q, k, v = (t.view(tokens, -1, dim) for t in merged.split([heads * dim, kv * dim, kv * dim], 1))
    slots = torch.randperm(pages * size, generator=g, device="cuda")[:tokens]
    slots[1::7] = -1
    slots[2::11] = pages * size + 3
    if tokens > 1:
        slots[-1] = pages * size
    slots = slots.to(torch.int32) if tokens % 2 else slots
    pos, table = torch.randint(0, 100000, (tokens,), generator=g, device="cuda"), ops.rotary_table(rot, interleaved=layout == "heads")
    y = ops.paged_append(k, v, keys, values, slots, positions=pos, table=table, query=q)
    rk = ops.rotary(k, pos, table).to(dtype)
    assert torch.equal(y, ops.rotary(q, pos, table))
    for cache, old, new in ((keys, before[0], rk), (values, before[1], v.to(dtype))):
        want = old.clone()
        rows = [(t, int(s)) for t, s in enumerate(slots.tolist()) if 0 <= s < pages * size]
        t, s = torch.tensor(rows, device="cuda").reshape(-1, 2).unbind(1)
        want[s // size, s % size] = new[t]
        assert torch.equal(cache, want)
    # without rotation; the query in place
    ops.paged_append(k, v, keys, values, slots)
    assert all(torch.equal(keys[s // size, s % size], k[t].to(dtype)) for t, s in rows[:50])
    want = ops.rotary(q, pos, table)
    assert ops.paged_append(k, v, keys, values, slots, positions=pos, table=table, query=q, out=q) is q and torch.equal(q, want)


# ---- attention ----------------------------------------------------------------------------------------------------
def _batch(g, lengths, new, kv, heads, dim, size, dtype, layout="rows", spare=3, poison=True):
    """(query, keys, values, pages, lengths, offsets): pages in any order; rows that hold no key are NaN, entries of the table
    behind a sequence's pages far outside."""
    used = [-(-max(n, 0) // size) for n in lengths]
    total = sum(used) + spare
    keys, values = _caches(g, total, size, kv, dim, dtype, layout)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(5)).tolist()
    pages = torch.full((len(lengths), max(used + [1]) + 1), 1 << 30, dtype=torch.int32)
    free = torch.ones(total, size, dtype=torch.bool)
    at = 0
    for i, n in enumerate(used):
        pages[i, :n] = torch.tensor(order[at:at + n])
        for j in range(n):
            free[order[at + j], :min(size, lengths[i] - j * size)] = False
        at += n
    if poison:
        for c in (keys, values):
            c[free.cuda()] = math.nan
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    query = _randn(g, offsets[-1], heads, dim, dtype=dtype)
    return query, keys, values, pages.cuda(), torch.tensor(lengths, device="cuda"), torch.tensor(offsets, device="cuda")


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,dim,size", [(4, 1, 128, 16), (6, 6, 64, 8), (10, 2, 72, 32), (16, 1, 128, 64), (40, 2, 96, 128), (3, 1, 8, 256)])
def test_one_new_token(dtype, heads, kv, dim, size):
    from glq_b200 import ops
    q, k, v, pages, lengths, offsets = _batch(_gen(heads), LENGTHS, [1] * len(LENGTHS), kv, heads, dim, size, dtype)
    y = ops.paged_attention(q, k, v, pages, lengths)
    ref, bound = O.attend(q, k, v, pages, lengths, offsets)
    _close(y, ref, bound)
    assert not y[0].any()
    assert torch.equal(y, ops.paged_attention(q, k, v, pages, lengths.to(torch.int32), query_offsets=offsets.to(torch.int32), max_query_len=1))


CHUNKS = {          # lengths, new tokens
    "one": ([300], [300]),
    "behind": ([1000], [77]),
    "mixed": ([0, 5, 130, 400, 64, 1, 700, 129], [0, 5, 1, 33, 64, 1, 2, 0]),
    "fewer keys than queries": ([3, 0, 70], [10, 4, 200]),
    "wide": ([600, 257], [513, 257]),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("mask", ["causal", "all", "window", "window of one", "all, window"])
@pytest.mark.parametrize("name", sorted(CHUNKS))
def test_chunks(dtype, mask, name):
    from glq_b200 import ops
    lengths, new = CHUNKS[name]
    causal, window = not mask.startswith("all"), {"window": 37, "window of one": 1, "all, window": 50}.get(mask, 0)
    for heads, kv, dim, size in ((4, 2, 128, 16), (5, 1, 64, 32)):
        q, k, v, pages, n, offsets = _batch(_gen(len(name)), lengths, new, kv, heads, dim, size, dtype)
        y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, causal=causal, window=window)
        ref, bound = O.attend(q, k, v, pages, n, offsets, causal=causal, window=window)
        _close(y, ref, bound, (heads, kv, dim, size))
        assert torch.equal(y, ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, causal=causal, window=window))


@pytest.mark.parametrize("new", [1, 3, 40, 200])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_query_does_not_see_changes_nothing(new, value):
    """Infinities and NaN in keys and values behind a query's own position, in front of its window."""
    from glq_b200 import ops
    lengths, news = [230, 200 + new], [new, new]
    q, k, v, pages, n, offsets = _batch(_gen(new), lengths, news, 2, 4, 128, 16, BF)
    clean = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, window=90)
    ref, bound = O.attend(q, k, v, pages, n, offsets, window=90)
    _close(clean, ref, bound)
    for i, bad in ((0, lengths[0] - 1), (0, 100), (1, lengths[1] - 1 - new // 2), (1, 3)):
        page = pages[i, bad // 16]
        kk, vv = k.clone(), v.clone()
        kk[page, bad % 16], vv[page, bad % 16] = value, value
        y = ops.paged_attention(q, kk, vv, pages, n, query_offsets=offsets, window=90)
        for r in range(2 * new):
            s, j = divmod(r, new)
            at = lengths[s] - new + j
            if s == i and at - 90 < bad <= at:
                assert not torch.isfinite(y[r].float()).all() or value == -math.inf
            else:
                assert torch.equal(y[r], clean[r]) or (y[r].double().cpu() - ref[r]).abs().le(bound[r]).all(), (i, bad, r)


def test_scores_without_a_softmax():
    """A visible key of minus infinity alone, plus infinity, NaN: as the definition has it, not a number."""
    from glq_b200 import ops
    q = torch.ones(1, 1, 64, device="cuda", dtype=HF)
    for value, length in ((-math.inf, 1), (math.inf, 5), (math.nan, 5)):
        k, v = torch.ones(1, 8, 1, 64, device="cuda", dtype=HF), torch.ones(1, 8, 1, 64, device="cuda", dtype=HF)
        k[0, 0] = value
        y = ops.paged_attention(q, k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([length], device="cuda"))
        assert torch.isnan(y).all(), value
    k[0, 0] = -math.inf                                                           # beside others: no weight
    assert torch.equal(ops.paged_attention(q, k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([5], device="cuda")), torch.ones_like(q))


@pytest.mark.parametrize("new", [1, 2, 150])
@pytest.mark.parametrize("layout", ["rows", "heads", "both"])
def test_layouts_strides_and_given_results(layout, new):
    from glq_b200 import ops
    lengths, news = [400, 150, 222], [new, new, new]
    q, k, v, pages, n, offsets = _batch(_gen(3), lengths, news, 2, 6, 96, 16, HF, layout)
    want, bound = O.attend(q, k, v, pages, n, offsets)
    y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets)
    _close(y, want, bound)
    for off, width in ((0, 600), (96, 800), (1, 577)):                             # rows of a merged projection, aligned and not
        buf = torch.zeros(3 * new + 1, width, device="cuda", dtype=HF).flatten()
        view = torch.as_strided(buf[off:], q.shape, (width, 96, 1))
        view.copy_(q)
        assert torch.equal(ops.paged_attention(view, k, v, pages, n, query_offsets=offsets), y)
        big = torch.full((3 * new + 1, width), 7.0, device="cuda", dtype=HF)
        out = torch.as_strided(big.flatten()[off:], q.shape, (width, 96, 1))
        assert ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, out=out) is out and torch.equal(out, y)
        out.fill_(7.0)
        assert bool((big == 7.0).all())
    assert torch.equal(ops.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, pages, n, query_offsets=offsets), y)
    table = torch.cat((pages, torch.full_like(pages, -1)), 1)[:, :pages.shape[1]]
    assert table.stride(0) != table.shape[1] and torch.equal(ops.paged_attention(q, k, v, table, n, query_offsets=offsets), y)
    half = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, scale=0.01)
    _close(half, *O.attend(q, k, v, pages, n, offsets, scale=0.01))


@pytest.mark.parametrize("rows", [60, 600])
def test_rows_of_no_sequence(rows):
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(1), [50, 90], [20, 20], 1, 2, 64, 16, BF)
    wide = torch.cat((q[:5], q, _randn(_gen(2), rows, 2, 64)))
    y = ops.paged_attention(wide, k, v, pages, n, query_offsets=offsets + 5)
    want = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets)
    assert torch.equal(y[5:45], want) and not y[:5].any() and not y[45:].any()
    out = torch.full_like(wide, 3.0)
    ops.paged_attention(wide, k, v, pages, n, query_offsets=offsets + 5, out=out)
    assert torch.equal(out[5:45], want) and bool((out[:5] == 3).all()) and bool((out[45:] == 3).all())
    empty = ops.paged_attention(wide, k, v, pages[:0], n[:0], query_offsets=offsets[:1])
    assert not empty.any()
    assert ops.paged_attention(q[:0], k, v, pages, n, query_offsets=offsets * 0).shape == (0, 2, 64)


@pytest.mark.parametrize("heads,kv,new", [(160, 1, 1), (160, 1, 3), (258, 2, 2), (128, 1, 5), (64, 1, 40), (7, 1, 100)])
def test_wide_groups_of_heads(heads, kv, new):
    """Up to 128 heads that share a key head are a tile's, more are the streaming kernel's."""
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(heads), [150, 70 + new], [new, new], kv, heads, 64, 16, HF)
    y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=new)
    _close(y, *O.attend(q, k, v, pages, n, offsets))


@pytest.mark.parametrize("new", [1, 3, 40])
def test_expanded_queries(new):
    from glq_b200 import ops
    _, k, v, pages, n, offsets = _batch(_gen(new), [90, 150], [new, new], 2, 4, 64, 16, BF)
    one = _randn(_gen(3), 1, 4, 64, dtype=BF)
    for q in (one.expand(2 * new, 4, 64), _randn(_gen(4), 2 * new, 1, 64, dtype=BF).expand(2 * new, 4, 64)):
        y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=new)
        ref, bound = O.attend(q, k, v, pages, n, offsets)
        _close(y, ref, bound)
        assert torch.equal(y, ops.paged_attention(q.contiguous(), k, v, pages, n, query_offsets=offsets, max_query_len=new))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [2, 60])
def test_windows_wider_than_any_sequence(new, causal):
    """Of sequences that are shorter than their queries too, where position - window is far below the first key."""
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(new), [1, new // 2, 300], [new] * 3, 2, 4, 64, 16, HF)
    want = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, causal=causal)
    _close(want, *O.attend(q, k, v, pages, n, offsets, causal=causal))
    for window in (400, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1):
        assert torch.equal(want, ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, causal=causal, window=window))


FIRST = """
import torch
from glq_b200 import ops
table = ops.rotary_table(64)
k, v = (torch.zeros(8, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
x = torch.randn(NEW, 8, 64, dtype=torch.bfloat16, device="cuda")
at = torch.arange(NEW, device="cuda")
pages = torch.arange(8, device="cuda", dtype=torch.int32)[None]
n, offsets = torch.tensor([NEW], device="cuda"), torch.tensor([0, NEW], device="cuda")
def step():
    q = ops.paged_append(x[:, 4:6], x[:, 6:], k, v, at, positions=at, table=table, query=x[:, :4])
    return ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=NEW)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = step()
graph.replay()
assert torch.equal(y, step()) and y.abs().sum() > 0
ops.check_device_status()
print("right")
"""


@pytest.mark.parametrize("new", [1, 100])
def test_first_call_of_a_process_is_captured(new):
    import subprocess
    import sys
    run = subprocess.run([sys.executable, "-c", FIRST.replace("NEW", str(new))], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert run.returncode == 0 and "right" in run.stdout, run.stderr[-2000:]


def test_no_pages_at_all():
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(3), [50, 90], [3, 40], 1, 2, 64, 16, BF)
    for longest in (1, 40):
        y = ops.paged_attention(q, k, v, pages[:, :0], n, query_offsets=offsets, max_query_len=longest)
        assert not y.any()


@pytest.mark.parametrize("longest", [0, 1, 4, 16, 300])
def test_bound_of_the_queries_changes_the_kernel_alone(longest):
    """max_query_len chooses the kernel; results are right whatever it says."""
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(8), [300, 40, 77], [130, 1, 20], 2, 8, 128, 32, BF)
    _close(ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=longest), *O.attend(q, k, v, pages, n, offsets))


@pytest.mark.parametrize("new", [1, 90])
def test_integers_that_make_no_sense_stay_in_bounds(new):
    """Pages outside the cache read as zeros, lengths are held to the table, offsets to the rows."""
    from glq_b200 import ops
    lengths = [200, 300]
    q, k, v, pages, n, offsets = _batch(_gen(4), lengths, [new, new], 1, 4, 128, 16, BF)
    bad = pages.clone()
    bad[0, 2], bad[0, 5], bad[1, 1] = -3, 10 ** 9, k.shape[0]
    _close(ops.paged_attention(q, k, v, bad, n, query_offsets=offsets), *O.attend(q, k, v, bad, n, offsets))
    most = bad.shape[1] * 16
    far = torch.tensor([2 ** 40, -5], device="cuda")
    _close(ops.paged_attention(q, k, v, bad, far, query_offsets=offsets), *O.attend(q, k, v, bad, torch.tensor([most, 0]), offsets))
    for wild in ([0, 10 ** 12, 2 * new], [-5, new, 10 ** 9], [2 * new, new, 0], [10 ** 9, -7, 3]):
        y = ops.paged_attention(q, k, v, pages, n, query_offsets=torch.tensor(wild, device="cuda"))
        assert y.shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("new", [1, 4])
def test_many_sequences(new):
    from glq_b200 import ops
    g = torch.Generator().manual_seed(8)
    lengths = (torch.randint(0, 90, (1500,), generator=g) + new).tolist()
    q, k, v, pages, n, offsets = _batch(_gen(6), lengths, [new] * 1500, 1, 2, 64, 16, BF, poison=False)
    _close(ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=new), *O.attend(q, k, v, pages, n, offsets))


def _reference(q, k, v, pages, length, scale):
    """One sequence, one token, in 64 bits on the device."""
    rows = k[pages].flatten(0, 1)[:length].double(), v[pages].flatten(0, 1)[:length].double()
    g = q.shape[1] // k.shape[2]
    z = torch.einsum("hd,nhd->hn", q[0].double(), rows[0].repeat_interleave(g, 1)) * scale
    return torch.einsum("hn,nhd->hd", torch.softmax(z, -1), rows[1].repeat_interleave(g, 1))


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 values, its last pages read and written."""
    from glq_b200 import ops
    pages, size, kv, dim = 140000, 32, 4, 128
    keys, values = (torch.zeros(pages, size, kv, dim, device="cuda", dtype=BF) for _ in range(2))
    assert keys.numel() > 2 ** 31
    ids = torch.tensor([[pages - 1, 0, pages - 2, 70000]], dtype=torch.int32, device="cuda")
    length = 100
    g = _gen(2)
    k, v, q = _randn(g, length, kv, dim), _randn(g, length, kv, dim), _randn(g, 1, 8, dim)
    at = torch.arange(length, device="cuda")
    ops.paged_append(k, v, keys, values, ids[0].long()[at // size] * size + at % size)
    assert torch.equal(keys[ids[0].long()].flatten(0, 1)[:length], k) and torch.equal(values[pages - 1], v[:size])
    y = ops.paged_attention(q, keys, values, ids, torch.tensor([length], device="cuda"))
    ref = _reference(q, keys, values, ids[0].long(), length, dim ** -0.5)
    assert (y[0].double() - ref).abs().max() <= 2.0 ** -7 * v.abs().max().double()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_long_context(dtype):
    from glq_b200 import ops
    size, length = 64, 70001
    g = _gen(9)
    n = -(-length // size)
    keys, values = _randn(g, n, size, 2, 128, dtype=dtype), _randn(g, n, size, 2, 128, dtype=dtype)
    pages = torch.randperm(n, generator=g, device="cuda").to(torch.int32)[None]
    q = _randn(g, 1, 8, 128, dtype=dtype) * 3
    y = ops.paged_attention(q, keys, values, pages, torch.tensor([length], device="cuda"))
    ref = _reference(q, keys, values, pages[0].long(), length, 128 ** -0.5)
    assert (y[0].double() - ref).abs().max() <= 2 * U[dtype] * values.abs().max().double()


def _reference_chunks(q, k, v, pages, lengths, offsets, window=0):
    """Attention in 64 bits on the device, a sequence and key head at a time."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    g = q.shape[1] // k.shape[2]
    for i, n in enumerate(lengths.tolist()):
        a, b = int(offsets[i]), int(offsets[i + 1])
        if a == b:
            continue
        ids = pages[i, :-(-n // k.shape[1])].long()
        at, key = torch.arange(n - (b - a), n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (key <= at) & ((key > at - window) if window else True)
        for h in range(k.shape[2]):
            z = torch.einsum("qgd,kd->gqk", q[a:b, h * g:(h + 1) * g].double(), k[ids][:, :, h].flatten(0, 1)[:n].double()) * q.shape[2] ** -0.5
            p = torch.softmax(torch.where(seen, z, -math.inf), -1)
            out[a:b, h * g:(h + 1) * g] = torch.einsum("gqk,kd->qgd", p, v[ids][:, :, h].flatten(0, 1)[:n].double())
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window", [0, 1500])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (15, 3, 64)])
@pytest.mark.parametrize("lengths,new", [([6000], [333]), ([2600], [2600]), ([5000, 17, 3000, 900, 2500, 64, 4000], [100, 17, 1, 300, 70, 1, 200])])
def test_long_chunks(dtype, window, heads, kv, dim, lengths, new):
    """Many key tiles per item, parts of items in several CTAs.  Values are normal: |out| <= max |v|, weights off by U each, the result by U."""
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(7), lengths, new, kv, heads, dim, 16, dtype, poison=False)
    ref = _reference_chunks(q, k, v, pages, n, offsets, window)
    for _ in range(3):
        y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, window=window)
        assert (y.double() - ref).abs().max() <= 2 * U[dtype] * v.abs().max().double()


# ---- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 72), (6, 2, 8), (5, 1, 120), (3, 3, 40), (20, 1, 96)])
@pytest.mark.parametrize("lengths,new", [([1700], [60]), ([900, 64, 1300, 5], [300, 1, 17, 5])])
def test_items_of_several_parts_in_heads_of_any_width(dtype, heads, kv, dim, lengths, new):
    """Results whose rows begin on 32 bytes, and in between."""
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(dim), lengths, new, kv, heads, dim, 16, dtype)
    ref, bound = O.attend(q, k, v, pages, n, offsets)
    y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets)
    _close(y, ref, bound)
    wide = torch.zeros(q.shape[0], heads, dim + 4, dtype=dtype, device="cuda")
    out = wide[:, :, :dim]
    ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, out=out)
    assert torch.equal(out, y) and not wide[:, :, dim:].any()


def test_prompt_then_decoding_steps():
    """A prompt in two chunks and decoding steps through append and attention, as a decoder runs them, against attention over the whole."""
    from glq_b200 import ops
    heads, kv, dim, size, steps = 8, 2, 128, 16, [40, 23, 1, 1, 1]
    g = _gen(11)
    total = sum(steps)
    qkv = _randn(g, total, (heads + 2 * kv) * dim)
    keys, values = (torch.full((9, size, kv, dim), math.nan, device="cuda", dtype=BF) for _ in range(2))
    pages = torch.tensor([[7, 2, 5, 0, 8, 1]], dtype=torch.int32, device="cuda")
    table = ops.rotary_table(dim, base=500000.0, scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    at = 0
    for n in steps:
        q, k, v = (t.view(n, -1, dim) for t in qkv[at:at + n].split([heads * dim, kv * dim, kv * dim], 1))
        pos = torch.arange(at, at + n, device="cuda")
        slots = pages[0].long()[pos // size] * size + pos % size
        rq = ops.paged_append(k, v, keys, values, slots, positions=pos, table=table, query=q)
        at += n
        offsets = torch.tensor([0, n], device="cuda")
        y = ops.paged_attention(rq, keys, values, pages, torch.tensor([at], device="cuda"), query_offsets=offsets, max_query_len=n)
        _close(y, *O.attend(rq, keys, values, pages, [at], offsets))


@pytest.mark.parametrize("new", [1, 130])
def test_captured_and_replayed_with_other_contents(new):
    """Two graphs of different batches over one cache, replayed in turn with other queries, lengths and pages in place."""
    from glq_b200 import ops
    batches = [_batch(_gen(s), lengths, [new] * len(lengths), 2, 8, 128, 16, BF) for s, lengths in ((1, [300, 200, 999]), (2, [777]))]
    graphs = []
    for q, k, v, pages, n, offsets in batches:
        call = lambda: ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=new)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
        graphs.append((graph, y))
    for step in range(3):
        for (q, k, v, pages, n, offsets), (graph, y) in zip(batches, graphs):
            q.copy_(_randn(_gen(50 + step), *q.shape))
            n.sub_(17)
            graph.replay()
        for (q, k, v, pages, n, offsets), (graph, y) in zip(batches, graphs):
            want = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, max_query_len=new)
            assert torch.equal(y, want)
            ref, bound = O.attend(q, k, v, pages, n, offsets)
            _close(y, ref, bound)


def test_calls_on_several_streams_at_once():
    from glq_b200 import ops
    work = [_batch(_gen(s), [500 + 40 * s, 900], [new, new], 2, 8, 128, 16, BF) for s, new in enumerate((1, 1, 64, 200))]
    want = [ops.paged_attention(q, k, v, p, n, query_offsets=o) for q, k, v, p, n, o in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, (q, k, v, p, n, o) in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(ops.paged_attention(q, k, v, p, n, query_offsets=o))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(0), [50, 60], [1, 1], 2, 4, 64, 16, BF)
    with pytest.raises(ValueError, match="over a cache"):
        ops.paged_attention(q.half(), k, v, pages, n)
    with pytest.raises(ValueError, match="overlaps"):
        ops.paged_attention(q, k, v, pages, n, out=q)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.paged_attention(q, k, v, pages.cpu(), n)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.paged_attention(q, k, v, pages, n.cpu())
    with pytest.raises(ValueError, match="16 bytes"):
        ops.paged_attention(q, torch.as_strided(k.flatten()[1:], (k.shape[0] - 1, *k.shape[1:]), k.stride()), v[:-1], pages, n)
    with pytest.raises(ValueError, match="overlaps the cache"):
        ops.paged_append(k[0], v[0], k, v, torch.zeros(16, dtype=torch.int64, device="cuda"))
    table = ops.rotary_table(64)
    with pytest.raises(ValueError, match="positions"):
        ops.rotary(q, torch.zeros(3, dtype=torch.int64, device="cuda"), table)
    with pytest.raises(ValueError, match="overlaps"):
        ops.rotary(q[:1], torch.zeros(1, dtype=torch.int64, device="cuda"), table, out=torch.as_strided(q, (1, 4, 64), (256, 64, 1), 8))


# ---- weights far below a row's largest ----------------------------------------------------------------------------
def _within(y, q, k, v, pages, lengths, offsets, window=0, what="", chain=None):
    """Each value against 64 bits on the device, within what its own weights allow.  A weight is rounded by U of itself or, of fp16's
    subnormal numbers, by half a step: weights are held as 2^7 times those relative to a score that is no larger than the row's
    largest, so 2^-25 is 2^-32 of the largest at most (bf16 has fp32's exponents).  The result is rounded by U of itself or, below 2^-14 in fp16, where
    numbers are multiples of 2^-24, by 2^-25.  In fp32: scores with
    `dim` products and sums, 2^-23 each where the tensor cores cut off, in a weight and in their sum; no sum is longer than the
    keys (or ``chain``), a step of it off by 2^-24 of what it has, in the values' sum and in the weights'."""
    g, dtype = q.shape[1] // k.shape[2], v.dtype
    floor, least = (2.0 ** -32, 2.0 ** -25) if dtype == HF else (0.0, 0.0)
    worst = -math.inf
    for i, n in enumerate(lengths.tolist()):
        a, b = int(offsets[i]), int(offsets[i + 1])
        ids = pages[i, :-(-n // k.shape[1])].long()
        at, key = torch.arange(n - (b - a), n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (key <= at) & ((key > at - window) if window else True)
        for h in range(k.shape[2]):
            kk, vv = (c[ids][:, :, h].flatten(0, 1)[:n].double() for c in (k, v))
            qq, own = q[a:b, h * g:(h + 1) * g].double(), y[a:b, h * g:(h + 1) * g].double()
            scale = q.shape[2] ** -0.5
            z = torch.where(seen, torch.einsum("qgd,kd->gqk", qq, kk) * scale, -math.inf)
            weight = torch.exp(z - z.amax(-1, keepdim=True))
            total = weight.sum(-1).transpose(0, 1)[..., None]
            ref, reach, far = (torch.einsum("gqk,kd->qgd", w, x) / total for w, x in ((weight, vv), (weight, vv.abs()), (seen.expand(g, -1, -1).double(), vv.abs())))
            size = torch.einsum("qgd,kd->gqk", qq.abs(), kk.abs()).masked_fill(~seen, 0.0).amax(-1).transpose(0, 1)[..., None] * scale
            fp32 = 2 * size * (q.shape[2] + 4) * 2.0 ** -23 + 2 * (chain or n) * 2.0 ** -24 + 2.0 ** -19
            bound = (U[dtype] + fp32) * reach + floor * far + U[dtype] * (ref.abs() + (U[dtype] + fp32) * reach + floor * far) + least
            worst = max(worst, float(((own - ref).abs() - bound).max()))
            assert bool(torch.isfinite(own).all()) and bool(((own - ref).abs() <= bound).all()), (what, i, h, worst)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("seqs", [1, 300])
@pytest.mark.parametrize("strong", [0, 70000, -10])
@pytest.mark.parametrize("below", [14.0, 20.0, 24.4, 25.4, 28.0])
def test_one_strong_key_and_many_weak_ones(dtype, new, seqs, strong, below):
    """One key has most of a row's weight and values of 0, 131,071 others 2^-below of it each and values of 1: theirs is the result, up to 0.9.
    Of one sequence each CTA has some keys, of 300 (that name the same pages) all or half of an item's."""
    from glq_b200 import ops
    n, dim, size = 131072, 64, 64
    k = torch.zeros(n // size, size, 1, dim, device="cuda", dtype=dtype)
    v = torch.ones_like(k)
    k.view(n, dim)[strong, 0] = below * math.log(2.0)
    v.view(n, dim)[strong] = 0.0
    q = torch.zeros(seqs * new, 4, dim, device="cuda", dtype=dtype)
    q[..., 0] = math.sqrt(dim)                                                     # (scores are the keys' first values)
    pages = torch.randperm(n // size, generator=_gen(1), device="cuda").to(torch.int32)[None]
    k[pages[0].long()], v[pages[0].long()] = k.clone(), v.clone()
    lengths, offsets = torch.full((seqs,), n, device="cuda"), torch.arange(seqs + 1, device="cuda") * new
    y = ops.paged_attention(q, k, v, pages.expand(seqs, -1), lengths, query_offsets=offsets, max_query_len=new)
    for i in sorted({0, 1 % seqs, seqs // 4, seqs // 2, seqs - 1}):
        mine = y[i * new:(i + 1) * new]
        _within(mine, q[:new], k, v, pages, lengths[:1], offsets[:2], what=(i, float(mine.float().mean())))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("above", [3.0, 7.9, 8.1, 15.9, 40.0])
def test_scores_that_grow_along_the_keys(dtype, new, above):
    """Later keys' weights are up to 2^above of the first one's: within the type, however far the reference lags behind."""
    from glq_b200 import ops
    n, dim = 5000, 64
    g = _gen(int(above))
    k, v = torch.zeros(1, 8192, 1, dim, device="cuda", dtype=dtype), _randn(g, 1, 8192, 1, dim, dtype=dtype)
    step = torch.where(torch.arange(8192, device="cuda") % 3000 < 1500, 0.0, above * math.log(2.0))
    k[0, :, 0, 0] = step.to(dtype)
    q = torch.zeros(new, 4, dim, device="cuda", dtype=dtype)
    q[..., 0] = math.sqrt(dim)
    pages, lengths, offsets = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([n], device="cuda"), torch.tensor([0, new], device="cuda")
    y = ops.paged_attention(q, k, v, pages, lengths, query_offsets=offsets, max_query_len=new)
    _within(y, q, k, v, pages, lengths, offsets)


def test_keys_and_values_in_one_place():
    """Attention may read one tensor as both; append may not write it as both."""
    from glq_b200 import ops
    q, k, _, pages, n, offsets = _batch(_gen(2), [50, 60], [1, 20], 2, 4, 64, 16, BF)
    _close(ops.paged_attention(q, k, k, pages, n, query_offsets=offsets), *O.attend(q, k, k, pages, n, offsets))
    new, slots, before = k[:1, 0].clone(), torch.zeros(1, dtype=torch.int64, device="cuda"), k.clone()
    for values in (k, torch.as_strided(k.flatten()[64:], (k.shape[0] - 1, *k.shape[1:]), k.stride())):
        with pytest.raises(RuntimeError, match="share addresses"):
            ops.paged_append(new, new, k[:len(values)], values, slots)
    assert torch.equal(k.nan_to_num(7.0), before.nan_to_num(7.0))


@pytest.mark.parametrize("dtype,dim", [(BF, 128), (HF, 64)])
def test_items_follow_one_another_in_a_ring(dtype, dim):
    """Each CTA of the streaming kernel has many items of every number of tiles, so that a ring's stages hold keys, then sums, then keys again."""
    from glq_b200 import ops
    seqs = 3000
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(1, 700, (seqs,), generator=g).tolist()
    q, k, v, _, n, offsets = _batch(_gen(5), [64 * 16], [seqs], 2, 8, dim, 16, dtype, poison=False)
    pages = torch.randint(0, k.shape[0], (seqs, 44), generator=g).to(torch.int32).cuda()
    lengths = torch.tensor(lengths, device="cuda")
    y = ops.paged_attention(q, k, v, pages, lengths)
    for _ in range(5):
        assert torch.equal(y, ops.paged_attention(q, k, v, pages, lengths))
    some = torch.arange(0, seqs, 37, device="cuda")
    _within(y[some], q[some], k, v, pages[some], lengths[some], torch.arange(len(some) + 1, device="cuda"))


@pytest.mark.parametrize("new", [3, 100])
def test_window_without_causal_begins_in_front_of_the_query(new):
    """Scores of 0: a query's result is the mean of the values from window - 1 keys in front of its own to the sequence's last."""
    from glq_b200 import ops
    n, window = 1000, 50
    k, v = torch.zeros(1, 1024, 1, 64, device="cuda", dtype=BF), torch.zeros(1, 1024, 1, 64, device="cuda", dtype=BF)
    pages, lengths, offsets = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([n], device="cuda"), torch.tensor([0, new], device="cuda")
    for key in (n - new - window, n - new - window + 1, n - window, n - 1):
        v.zero_()
        v[0, key] = 1.0
        y = ops.paged_attention(torch.ones(new, 8, 64, device="cuda", dtype=BF), k, v, pages, lengths, query_offsets=offsets, causal=False, window=window)
        for i, at in enumerate(range(n - new, n)):
            first = at - window + 1
            want = 1.0 / (n - first) if key >= first else 0.0
            assert (y[i].double() - want).abs().max() <= 2.0 ** -7 * want, (i, key)


def _told_apart(v, pages, size):
    """Values (pages, rows, heads, dim) that are 0 but in one column, which 64 keys of a sequence have in turn: the results' columns say what each 64 keys gave, and one
    that is lost or counted twice is an eighth of a column at least of 70,000 keys, where bounds are a hundredth."""
    key = torch.arange(pages.numel() * size, device=v.device)
    column = torch.zeros(v.shape[0] * size, dtype=torch.long, device=v.device)
    column[pages.long().flatten()[key // size] * size + key % size] = key // 64 % v.shape[3]
    only = (column[:, None] == torch.arange(v.shape[3], device=v.device)).view(v.shape[0], size, 1, -1)
    return ((v.abs() + 0.5) * only).to(v.dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kv,group,new", [(2, 4, 1), (1, 2, 1), (2, 4, 20)])
def test_long_context_value_by_value(dtype, kv, group, new):
    """148 CTAs at least have a share each: 2 * 70,001 keys are less than 1024 for one, and as many parts as
    CTAs are joined."""
    from glq_b200 import ops
    size, length = 64, 70001
    g = _gen(19)
    n = -(-length // size)
    keys, values = _randn(g, n, size, kv, 128, dtype=dtype), _randn(g, n, size, kv, 128, dtype=dtype)
    pages = torch.randperm(n, generator=g, device="cuda").to(torch.int32)[None]
    q, values = _randn(g, new, kv * group, 128, dtype=dtype), _told_apart(values, pages, size)
    lengths, offsets = torch.tensor([length], device="cuda"), torch.tensor([0, new], device="cuda")
    y = ops.paged_attention(q, keys, values, pages, lengths, query_offsets=offsets, max_query_len=new)
    _within(y, q, keys, values, pages, lengths, offsets, chain=1024 + 296)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window", [0, 1500])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (15, 3, 64)])
@pytest.mark.parametrize("lengths,new", [([6000], [333]), ([2600], [2600]), ([5000, 17, 3000, 900, 2500, 64, 4000], [100, 17, 1, 300, 70, 1, 200])])
def test_long_chunks_value_by_value(dtype, window, heads, kv, dim, lengths, new):
    from glq_b200 import ops
    q, k, v, pages, n, offsets = _batch(_gen(17), lengths, new, kv, heads, dim, 16, dtype, poison=False)
    for i, length in enumerate(lengths):
        mine = pages[i, :-(-length // 16)]
        v[mine.long()] = _told_apart(v, mine, 16)[mine.long()]
    y = ops.paged_attention(q, k, v, pages, n, query_offsets=offsets, window=window)
    _within(y, q, k, v, pages, n, offsets, window)


WITHOUT_CHAINING = """
import torch
from glq_b200 import ops
g = torch.Generator(device="cuda").manual_seed(3)
rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
table, k, v = ops.rotary_table(64), rand(40, 16, 2, 64), rand(40, 16, 2, 64)
pages = torch.randperm(40, generator=g, device="cuda").to(torch.int32)[None]
for new, total in ((200, 200), (1, 201), (40, 241), (1, 242)):
    x, at = rand(new, 8, 64), torch.arange(total - new, total, device="cuda")
    q = ops.paged_append(x[:, 4:6], x[:, 6:], k, v, pages[0].long()[at // 16] * 16 + at % 16, positions=at, table=table, query=x[:, :4])
    assert torch.equal(q, ops.rotary(x[:, :4], at, table))
    y = ops.paged_attention(q, k, v, pages, torch.tensor([total], device="cuda"), query_offsets=torch.tensor([0, new], device="cuda"), max_query_len=new)
    print(new, y.view(torch.int16).long().sum().item(), k.view(torch.int16).long().sum().item())
ops.check_device_status()
"""


def test_launches_that_are_not_chained():
    """GLQB_PDL=0, which is read once in a process: the same bits."""
    import subprocess
    import sys
    said = []
    for value in ("1", "0"):
        run = subprocess.run([sys.executable, "-c", WITHOUT_CHAINING], capture_output=True, text=True, timeout=300, env={**os.environ, "GLQB_PDL": value},
                             cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
        assert run.returncode == 0, run.stderr[-2000:]
        said.append(run.stdout)
    assert said[0] == said[1] and said[0].count("\n") == 4
