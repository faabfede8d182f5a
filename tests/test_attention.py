"""Attention over the paged cache - cybq_attention - against its definition in float64.

Bound of an output element, S = sum of p |v| over what its row sees, D = the largest sum of |q| |k| scale:
  y's own rounding       half a step of its type, of y
  values, Q8 and Q4      round_f16(scale q): 2^-11 S;   P of f16: 2^-11 S;   P of bf16 as two numbers: 2^-16 S, as one (many rows): 2^-8 S
  scores                 products are exact, a sum of `dim` of them and its scales in fp32: (dim + 8) 2^-24 D absolute, of keys rounded to
                         f16 (many rows on Q8, Q4) 2^-11 D more; the exponent's argument and the exponential 2^-21 more for scores up to 4;
                         a score's error is a relative one of its P, and of the sum that divides: twice
  sums                   fp32, at most a few hundred terms in a row before others join: 2^-15 S
  quantised, bf16 q      a row becomes f16 behind a power of two: exact but for what is 2^-25 of its largest, below the terms above"""
import math

import numpy as np
import pytest

from cyb_amd.backend import Backend

torch = pytest.importorskip("torch")
from tests.cache_lib import HALF_STEP, TDT, Cached, normal, rope_table      # noqa: E402

gpu = pytest.mark.gpu
U = 2.0 ** -24
FEW = 64                # rows of a sequence and kv head (new tokens times group); "many rows" above are more than these


def bound(kind, dt, dim, y, size, dots, many):
    quantised = kind in ("q8", "q4")
    p = 2.0 ** -11 if kind != "bf16" else 2.0 ** -8 if many else 2.0 ** -16
    score = (dim + 8) * U * dots + 2.0 ** -21 + (2.0 ** -11 * dots if quantised and many else 0.0)
    return HALF_STEP[dt] * y.abs() + size * (p + (2.0 ** -11 if quantised else 0.0) + 2 * score + 2.0 ** -15) + 2.0 ** -25


def check(s, new, group, dt, window=0, many=False, scale=None, hidden=lambda b, j: False, rows=None, stream=0, q=None, seed=9):
    rows = rows if rows is not None else sum(new)
    q = q if q is not None else normal((rows, s.kv_heads * group, s.dim), seed, dt)
    y = torch.full((rows,) + tuple(q.shape[1:]), 9.0, dtype=TDT[dt], device="cuda")
    s.be.attention(s.cache, s.layer, s.batch(new, rows=rows), q, y, scale=scale, window=window, stream=stream)
    torch.cuda.synchronize()
    used = sum(new)
    ref, size, dots = s.expected(q[:used], new, scale, window, hidden)
    assert torch.isfinite(y).all()
    off = (y[:used].double() - ref).abs()
    many = many or max(new) * group > FEW
    worst = (off / bound(s.kind, dt, s.dim, ref, size, dots, many)).max().item() if used else 0.0
    assert worst <= 1.0, worst
    assert (y[used:] == 9.0).all()                               # rows of no sequence
    return y


KINDS = [("f16", "f16"), ("bf16", "bf16"), ("q8", "f16"), ("q8", "bf16"), ("q4", "f16"), ("q4", "bf16")]


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_one_token_of_every_length(backend, kind, dt, dim):
    lengths = [1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 300, 511, 777]
    s = Cached(backend, kind, lengths, kv_heads=2, dim=dim, page=64)
    for group in (1, 4, 7):
        check(s, [1] * len(lengths), group, dt)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("page", [32, 256, 1024])
def test_drafts_and_windows(backend, kind, dt, page):
    """A few new rows each: rows that see different tokens, more than a tile of them, windows that begin and end anywhere."""
    lengths, new = [5, 40, 300, 1030, 64], [5, 3, 7, 2, 4]
    s = Cached(backend, kind, lengths, kv_heads=2, dim=128, page=page)
    for group in (1, 3, 5, 16):
        for window in (0, 1, 2, 31, 32, 33, 200, 5000):
            check(s, new, group, dt, window=window)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_prompts(backend, kind, dt, dim):
    """Hundreds of rows: from a prompt's first token on, and behind what is cached."""
    for lengths, new, window in (([200], [200], 0), ([333, 150, 700], [100, 150, 391], 0), ([600], [300], 100), ([513], [129], 0)):
        s = Cached(backend, kind, lengths, kv_heads=1, dim=dim, page=64, seed=len(lengths))
        check(s, new, 3, dt, window=window, many=True)
        s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
def test_prompts_exactly(backend, kind, dt):
    """Many rows with the prefill mode EXACT: the bound of few."""
    backend.set_prefill_mode("exact")
    try:
        for lengths, new, window, dim in (([333, 150, 700], [100, 150, 391], 0, 128), ([600], [300], 100, 64), ([513], [129], 0, 256)):
            s = Cached(backend, kind, lengths, kv_heads=2, dim=dim, page=64, seed=len(lengths))
            q = normal((sum(new), 6, dim), 9, dt)
            y = torch.empty_like(q)
            backend.attention(s.cache, 0, s.batch(new), q, y, window=window)
            torch.cuda.synchronize()
            ref, size, dots = s.expected(q, new, None, window)
            worst = ((y.double() - ref).abs() / bound(kind, dt, dim, ref, size, dots, False)).max().item()
            assert worst <= 1.0, worst
            s.close()
    finally:
        backend.set_prefill_mode("fast")


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
def test_a_long_context_is_shared_out(backend, kind, dt):
    s = Cached(backend, kind, [20011, 130], kv_heads=2, dim=128, page=128)
    check(s, [1, 1], 4, dt)
    check(s, [3, 2], 5, dt, window=15000)
    s.close()


@gpu
def test_more_sequences_than_lanes(backend):
    rng = np.random.default_rng(2)
    lengths = rng.integers(0, 200, 200).tolist()
    lengths[100], lengths[3] = 6000, 0
    s = Cached(backend, "q8", lengths, kv_heads=2, dim=64, page=32)
    new = [min(L, int(n)) for L, n in zip(lengths, rng.integers(0, 4, 200))]
    check(s, new, 3, "f16", rows=sum(new) + 5)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", [("f16", "f16"), ("q4", "bf16")])
def test_rows_that_see_nothing(backend, kind, dt):
    """Sequences without tokens, more rows than tokens, pages that are none, a whole window without a page: zeros, never NaN."""
    s = Cached(backend, kind, [96, 40, 300], kv_heads=2, dim=64, page=32)
    s.tables[0, 0] = -1
    s.tables[2, 3:8] = 1 << 30                                    # tokens 96 .. 255 are in no page
    group = 2
    # rows 0 .. 31 of the first sequence see nothing
    y = check(s, [96, 1, 60], group, dt, hidden=lambda b, j: (b == 0 and j < 32) or (b == 2 and 96 <= j < 256), many=True)
    assert (y[:32] == 0).all()
    y = check(s, [1, 1, 50], group, dt, window=10, hidden=lambda b, j: (b == 0 and j < 32) or (b == 2 and 96 <= j < 256))
    assert (y[2:8] == 0).all()                                   # positions 250 .. 255 with a window of 10
    # a length that the rows exceed, and none at all
    q = normal((12, 4, 64), 3, dt)
    out = torch.full_like(q, 9.0)
    backend.attention(s.cache, 0, s.batch([7, 5, 0], lengths=[3, 0, 0]), q, out)
    torch.cuda.synchronize()
    assert (out[:4] == 0).all() and (out[7:] == 0).all() and torch.isfinite(out).all()
    s.close()


@gpu
def test_values_at_the_ends(backend):
    """Scores that differ by thousands, equal ones, a scale of the caller's, keys and values at the ends of the kinds, rows of NaN."""
    for kind, dt in KINDS:
        s = Cached(backend, kind, [100], kv_heads=1, dim=64, page=32)
        q = normal((4, 2, 64), 1, dt) * 100
        check(s, [4], 2, dt, q=q, scale=0.5)                     # one token has it all
        check(s, [4], 2, dt, q=torch.zeros_like(q))              # the mean
        check(s, [4], 2, dt, scale=1e-6)
        q[1, 0, 5] = math.nan
        y = torch.empty_like(q)
        backend.attention(s.cache, 0, s.batch([4]), q, y)
        torch.cuda.synchronize()
        bad = torch.isnan(y).all(dim=2)
        assert bad[1, 0] and bad.sum() == 1 and torch.isnan(y).sum() == 64
        s.close()
    # rows of bf16 far outside f16 on a quantised cache
    s = Cached(backend, "q8", [50], kv_heads=1, dim=64, page=32)
    check(s, [2], 2, "bf16", q=normal((2, 2, 64), 2, "bf16", std=1e25), scale=1e-25)
    check(s, [2], 2, "bf16", q=normal((2, 2, 64), 2, "bf16", std=1e-25), scale=1e25)
    s.close()
    # infinities and NaN that were stored are finite numbers: no other row meets them
    for kind, dt in KINDS:
        s = Cached(backend, kind, [64], kv_heads=1, dim=64, page=32)
        x = normal((2, 1, 64), 4, dt)
        x[1] = math.inf
        x[1, 0, 3] = math.nan
        backend.cache_append(s.cache, 0, s.batch([2]), None, normal((2, 1, 64), 5, dt), x)
        q = normal((2, 1, 64), 6, dt)
        y, first = torch.empty_like(q), torch.empty_like(q)
        backend.attention(s.cache, 0, s.batch([2]), q, y)
        backend.cache_append(s.cache, 0, s.batch([2]), None, normal((2, 1, 64), 5, dt), torch.where(torch.isfinite(x), x, 0.0))
        backend.attention(s.cache, 0, s.batch([2]), q, first)
        torch.cuda.synchronize()
        assert torch.equal(y[0], first[0])
        s.close()


@gpu
def test_strides_streams_and_the_same_bits_twice(backend):
    """q as a slice of the projection's rows, on a stream of its own; results do not hang on who arrives first."""
    s = Cached(backend, "q8", [3000, 1500], kv_heads=2, dim=128, page=64)
    wide = normal((5, 6 * 4, 128), 7, "f16")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    a = check(s, [3, 2], 4, "f16", q=wide[:, 8:16], stream=side.cuda_stream)
    for _ in range(3):
        assert torch.equal(a, check(s, [3, 2], 4, "f16", q=wide[:, 8:16].contiguous()))
    s.close()


@gpu
def test_a_captured_step_follows_its_lengths(backend):
    """Append and attention recorded once, on a fresh context; replayed with other lengths, tables and rows, with eager calls in between."""
    be = Backend(0)
    try:
        B, group, page, width, dim = 3, 4, 32, 100, 64
        s = Cached(be, "q8", [700, 40, 2900], kv_heads=2, dim=dim, page=page, width=width, spare=40)
        rope = rope_table(width * page, dim)
        qkv = normal((B, (group + 2) * 2, dim), 11, "f16")
        q, y = (torch.zeros((B, group * 2, dim), dtype=torch.float16, device="cuda") for _ in range(2))
        starts = torch.arange(B + 1, dtype=torch.int32, device="cuda")
        lengths = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
        batch = be.cache_batch(starts, lengths, s.tables, B, 1)

        def step(stream=0):
            h = group * 2
            be.cache_append(s.cache, 0, batch, qkv[:, :h], qkv[:, h:h + 2], qkv[:, h + 2:], q, rope=rope, stream=stream)
            be.attention(s.cache, 0, batch, q, y, window=2000, stream=stream)

        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            step(torch.cuda.current_stream().cuda_stream)
        for i, now in enumerate(([700, 40, 2900], [1, 39, 2], [512, 1, 2899], [700, 40, 2900])):
            lengths.copy_(torch.tensor(now, dtype=torch.int32))
            qkv.copy_(normal(tuple(qkv.shape), 20 + i, "f16"))
            y.zero_()
            q.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got, turned_q = y.clone(), q.clone()
            y.zero_()
            q.zero_()
            step()
            torch.cuda.synchronize()
            assert torch.equal(got, y) and torch.equal(turned_q, q) and (got != 0).any()
        s.close()
    finally:
        be.close()


@gpu
def test_batches_that_make_no_sense_stay_inside(backend):
    """Starts that fall or lie outside, lengths below zero and beyond the table: some rows, no access outside (checked in the kernels)."""
    s = Cached(backend, "q8", [64, 64, 64], kv_heads=1, dim=64, page=32)
    q = normal((8, 2, 64), 1, "f16")
    guard = torch.full((24, 2, 64), 9.0, dtype=torch.float16, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for starts, lengths in (([0, 8, 0, 8], [64, 64, 64]), ([-5, 3, 100, 2], [64, 64, 64]), ([0, 1 << 30, -(1 << 30), 8], [1 << 30, -7, 64]),
                            ([0, 2, 4, 8], [-(1 << 31), (1 << 31) - 1, 70])):
        b = backend.cache_batch(ints(starts), ints(lengths), s.tables, 8, 8)
        y = guard[8:16]
        backend.attention(s.cache, 0, b, q, y)
        backend.cache_read(s.cache, 0, b, torch.empty((8, 1, 64), device="cuda"), torch.empty((8, 1, 64), device="cuda"))
        torch.cuda.synchronize()
        assert (guard[:8] == 9.0).all() and (guard[16:] == 9.0).all()
    check(s, [3, 1, 2], 2, "f16")                                # and what comes after is right
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", [("f16", "f16"), ("bf16", "bf16"), ("q8", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_many_rows_of_a_long_context(backend, kind, dt, dim):
    """Parts of more blocks than a register of pages has, pages that are missing among them, next to single tokens and a short prompt."""
    lengths, new, group, page = [5000, 300, 40, 2100], [515, 1, 1, 100], 4, 32
    s = Cached(backend, kind, lengths, kv_heads=4, dim=dim, page=page, seed=dim)
    s.tables[0, 70], s.tables[0, 129], s.tables[3, 5] = -1, s.cache.pages, -7
    hidden = lambda b, j: (b == 0 and j // page in (70, 129)) or (b == 3 and j // page == 5)
    y = check(s, new, group, dt, hidden=hidden)
    assert torch.equal(y, check(s, new, group, dt, hidden=hidden))
    check(s, new, group, dt, window=2300, hidden=hidden)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt,dim", [("f16", "f16", 128), ("bf16", "bf16", 64), ("q8", "f16", 128), ("q4", "bf16", 96), ("f16", "f16", 256)])
def test_tiles_that_are_not_cut(backend, kind, dt, dim):
    """As many tiles as there are workgroups, each with all of its blocks (150 of the last); odd rows in the last."""
    s = Cached(backend, kind, [4800], kv_heads=8, dim=dim, page=256)
    check(s, [1027 if dim > 64 else 2051], 4, dt)
    s.close()


@gpu
def test_pages_past_4_gib(backend):
    """A page whose bytes lie more than 2^32 behind the cache's first, few rows and many; and the caller's copy of it elsewhere."""
    page, pages = 1024, 1100
    cache = backend.kv_cache("f16", 1, 8, 128, page, pages)
    assert cache.page_bytes * pages > 1 << 32
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    n = 1500
    k, v = normal((n, 8, 128), 1, "f16"), normal((n, 8, 128), 2, "f16")
    q = normal((n, 16, 128), 3, "f16")
    outs = []
    for table in ([pages - 1, 1050], [0, 1]):
        b = backend.cache_batch(ints([0, n]), ints([n]), ints([table]), n)
        backend.cache_append(cache, 0, b, None, k, v)
        k2, v2 = torch.empty_like(k), torch.empty_like(v)
        backend.cache_read(cache, 0, b, k2, v2)
        few = backend.cache_batch(ints([0, 3]), ints([n]), ints([table]), 3)
        y, y3 = torch.empty_like(q), torch.empty_like(q[:3])
        backend.attention(cache, 0, b, q, y)
        backend.attention(cache, 0, few, q[n - 3:], y3)
        torch.cuda.synchronize()
        assert torch.equal(k2, k) and torch.equal(v2, v)
        outs.append((y, y3))
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and (outs[0][0] != 0).any()
    cache.free()


@gpu
def test_a_captured_prompt(backend):
    """Many rows next to few in a graph, replayed with other lengths with eager calls of other shapes in between; a context of its own."""
    be = Backend(0)
    try:
        s = Cached(be, "q8", [900, 2000, 60], kv_heads=2, dim=128, page=64, width=40)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        starts, lengths = ints([0, 600, 601, 604]), ints([900, 2000, 60])
        batch = be.cache_batch(starts, lengths, s.tables, 604, 2000)
        q = normal((604, 20, 128), 5, "f16")
        y = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            be.attention(s.cache, 0, batch, q, y, stream=torch.cuda.current_stream().cuda_stream)
        for st, ln in (([0, 600, 601, 604], [900, 2000, 60]), ([0, 1, 602, 604], [900, 1999, 60]), ([0, 3, 6, 9], [5, 1200, 60]), ([0, 600, 601, 604], [600, 64, 3])):
            starts.copy_(ints(st))
            lengths.copy_(ints(ln))
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            check(s, [2, 1, 3], 4, "f16", rows=7)
            y.zero_()
            be.attention(s.cache, 0, batch, q, y)
            torch.cuda.synchronize()
            assert torch.equal(got, y) and (got[:st[-1]] != 0).any() and (got[st[-1]:] == 0).all()
        s.close()
    finally:
        be.close()


@gpu
def test_two_contexts_on_one_cache(backend):
    """Another context appends to and reads pages of its own, on a stream of its own, while the first attends to others."""
    other = Backend(0)
    try:
        s = Cached(backend, "q8", [3000, 800], kv_heads=2, dim=128, page=64, spare=20)
        free = sorted(set(range(s.cache.pages)) - set(s.tables.flatten().tolist()))
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        k, v = normal((500, 2, 128), 1, "f16"), normal((500, 2, 128), 2, "f16")
        q = normal((500, 8, 128), 3, "f16")
        b = other.cache_batch(ints([0, 500]), ints([500]), ints([free[:8]]), 500)
        want = torch.empty_like(q)
        backend.cache_append(s.cache, 0, b, None, k, v)
        backend.attention(s.cache, 0, b, q, want)
        side = torch.cuda.Stream()
        first = check(s, [4, 3], 4, "f16")
        mine = normal((7, 8, 128), 9, "f16")
        got, y = torch.empty_like(q), torch.empty_like(mine)
        batch = s.batch([4, 3])
        torch.cuda.synchronize()
        for _ in range(20):
            other.cache_append(s.cache, 0, b, None, k, v, stream=side.cuda_stream)
            other.attention(s.cache, 0, b, q, got, stream=side.cuda_stream)
            backend.attention(s.cache, 0, batch, mine, y)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(y, first)
        s.close()
    finally:
        other.close()


@gpu
def test_many_rows_of_batches_that_make_no_sense(backend):
    """As above for calls of many rows; rows outside of the call's stay as they were."""
    s = Cached(backend, "bf16", [2000, 64, 64], kv_heads=8, dim=64, page=32)
    q = normal((1000, 32, 64), 1, "bf16")
    guard = torch.full((1400, 32, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for starts, lengths in (([0, 1000, 0, 1000], [2000, 64, 64]), ([-5, 3, 4000, 2], [2000, 64, 64]), ([0, 1 << 30, -(1 << 30), 1000], [1 << 30, -7, 64]),
                            ([0, 200, 600, 1000], [-(1 << 31), (1 << 31) - 1, 70])):
        b = backend.cache_batch(ints(starts), ints(lengths), s.tables, 1000, 1000)
        backend.attention(s.cache, 0, b, q, guard[200:1200])
        torch.cuda.synchronize()
        assert (guard[:200] == 9.0).all() and (guard[1200:] == 9.0).all()
    check(s, [900, 1, 2], 4, "bf16")
    s.close()


@gpu
@pytest.mark.parametrize("rows", [3, 300])
def test_the_plain_binding_gives_the_same(backend, monkeypatch, rows):
    """Without the native call path: the same bits, the same refusals; a cache that was freed is refused by both."""
    from cyb_amd import backend as module
    from cyb_amd.backend import CybqError
    s = Cached(backend, "q8", [rows + 50], kv_heads=2, dim=64, page=32)
    wide, rope = normal((rows, 8, 64), 3, "f16"), rope_table(s.tables.shape[1] * 32, 64)
    outs = []

    def status(call):
        with pytest.raises(CybqError) as e:
            call()
        return e.value.status

    for native in (True, False):
        if not native:
            monkeypatch.setattr(module, "_calls", False)
        batch, q = s.batch([rows]), torch.empty((rows, 4, 64), dtype=torch.float16, device="cuda")
        y, k, v = torch.empty_like(q), torch.empty((rows, 2, 64), device="cuda"), torch.empty((rows, 2, 64), device="cuda")
        backend.cache_append(s.cache, 0, batch, wide[:, :4], wide[:, 4:6], wide[:, 6:], q, rope=rope, style="pairs")
        backend.cache_read(s.cache, 0, batch, k, v)
        backend.attention(s.cache, 0, batch, q, y, scale=0.2, window=40)
        torch.cuda.synchronize()
        refused = [status(lambda: backend.attention(s.cache, 1, batch, q, y)), status(lambda: backend.attention(s.cache, 0, batch, q[:, :3], y[:, :3])),
                   status(lambda: backend.attention(s.cache, 0, batch, q, y.float())), status(lambda: backend.attention(s.cache, 0, batch, q, y, scale=-1.0)),
                   status(lambda: backend.attention(s.cache, 0, batch, q, y, window=-1)), status(lambda: backend.attention(s.cache, 0, batch, q[:rows - 1], y)),
                   status(lambda: backend.attention(s.cache, 0, batch, q, y.cpu())), status(lambda: backend.cache_read(s.cache, 0, batch, k, v[:, :1])),
                   status(lambda: backend.cache_append(s.cache, 0, batch, None, k, v.half())), status(lambda: backend.cache_append(s.cache, 0, batch, wide[:, :4], k, v)),
                   status(lambda: backend.cache_append(s.cache, 0, batch, None, k, v, rope=rope[:32]))]
        gone = backend.kv_cache("q8", 1, 2, 64, 32, 4)
        gone.free()
        refused.append(status(lambda: backend.cache_read(gone, 0, batch, k, v)))
        outs.append((q, y, k, v, refused))
    assert all(torch.equal(a, b) for a, b in zip(outs[0][:4], outs[1][:4])) and outs[0][4] == outs[1][4] and 0 not in outs[0][4]
    s.close()


@gpu
def test_nothing_to_do(backend):
    """No sequences, no rows, sequences without new rows: nothing is written, and nothing refused."""
    s = Cached(backend, "f16", [64, 64], kv_heads=1, dim=64, page=32)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    y = torch.full((4, 2, 64), 9.0, dtype=torch.float16, device="cuda")
    k = torch.full((4, 1, 64), 9.0, dtype=torch.float16, device="cuda")
    for b in (backend.cache_batch(ints([0]), ints([]), s.tables[:0], 4), backend.cache_batch(ints([0, 0, 0]), ints([64, 64]), s.tables, 0),
              backend.cache_batch(ints([0, 0, 0]), ints([64, 64]), s.tables, 4), backend.cache_batch(ints([0, 0, 0]), ints([64, 64]), s.tables, 4, 1000)):
        backend.cache_append(s.cache, 0, b, torch.zeros_like(y), torch.zeros_like(k), torch.zeros_like(k), y)
        backend.cache_read(s.cache, 0, b, k, k.clone())
        backend.attention(s.cache, 0, b, torch.zeros_like(y), y)
        torch.cuda.synchronize()
        assert (y == 9.0).all() and (k == 9.0).all()
    check(s, [2, 1], 2, "f16")
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
def test_one_kv_head_for_hundreds(backend, kind, dt):
    """Groups wider than a tile of either kernel, so that a token's heads are several tiles."""
    s = Cached(backend, kind, [700, 90], kv_heads=1, dim=64, page=32)
    for group in (71, 600):
        check(s, [1, 2], group, dt)
    s.close()


@gpu
@pytest.mark.parametrize("new", [3, 200])
def test_factors_that_vanish(backend, new):
    """Rows and scales so small that a score's factor is below fp32: every token weighs the same, and hidden ones nothing."""
    for kind in ("q8", "q4", "bf16"):
        s = Cached(backend, kind, [300], kv_heads=1, dim=64, page=32)
        q = normal((new, 4, 64), 2, "bf16", std=1e-30)
        check(s, [new], 4, "bf16", q=q, scale=1e-25, window=100)
        check(s, [new], 4, "bf16", q=normal((new, 4, 64), 2, "bf16"), scale=1e-44, window=100)
        s.close()
