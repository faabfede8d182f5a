"""Attention over the paged cache in calls whose sizes say little about their rows, with scores of any
size, probabilities and values far apart.  Against float64; the bound of an element is that of test_attention.py."""
import math

import pytest

torch = pytest.importorskip("torch")
from tests.cache_lib import TDT, Cached, held, normal      # noqa: E402
from tests.test_attention import FEW, KINDS, bound, check  # noqa: E402

gpu = pytest.mark.gpu


def check_each(s, new, group, dt, window=0, scale=None, rows=None, max_new=None, q=None, seed=9, exact=False, unit=1.0, exact_scores=False):
    """As `check`, each sequence against the bound of its own number of rows (exact: of few), values counted in `unit`.  Scores of any size: what
    the exponent's argument and the factors that scale sums anew lose, at most 4 U of the largest score, is counted as four dimensions more; exact_scores:
    they are equal or far apart, and nothing is lost."""
    rows = sum(new) if rows is None else rows
    q = normal((rows, s.kv_heads * group, s.dim), seed, dt) if q is None else q
    y = torch.full(q.shape, 9.0, dtype=TDT[dt], device="cuda")
    s.be.attention(s.cache, s.layer, s.batch(new, rows=rows, max_new=max_new), q, y, scale=scale, window=window)
    torch.cuda.synchronize()
    used = sum(new)
    ref, size, dots = s.expected(q[:used], new, scale, window)
    dots = dots * (0.0 if exact_scores else 1.0)
    many = torch.tensor([n * group > FEW and not exact for n in new for _ in range(n)], device="cuda").reshape(-1, 1, 1)
    most = torch.where(many, *(bound(s.kind, dt, s.dim + 4, ref / unit, size / unit, dots, m) * unit for m in (True, False)))
    assert torch.isfinite(y[:used]).all()
    worst = ((y[:used].double() - ref).abs() / most).max().item()
    assert worst <= 1.0, worst
    assert (y[used:] == 9.0).all()
    return y


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
def test_one_sequence_is_what_its_rows_make_it(backend, kind, dt):
    """A few rows of the only sequence of a call, with a max_new and rows of padding that would hold a prompt: the exact kernel's bits and bound."""
    s = Cached(backend, kind, [300], kv_heads=2, dim=128, page=64)
    for new in (1, 3):
        tight = check_each(s, [new], 4, dt)
        for rows, max_new in ((new, 4096), (new + 5, 4096), (700, 700), (700, 1 << 24)):
            q = normal((rows, 8, 128), 9, dt)
            q[:new] = normal((new, 8, 128), 9, dt)
            assert torch.equal(check_each(s, [new], 4, dt, rows=rows, max_new=max_new, q=q)[:new], tight)
    check_each(s, [200], 4, dt, rows=210, max_new=4096)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
def test_each_sequence_of_a_mixed_call_has_its_own_bound(backend, kind, dt):
    s = Cached(backend, kind, [900, 300, 40, 700], kv_heads=8, dim=64, page=64)
    check_each(s, [400, 1, 5, 16], 4, dt, rows=430)
    s.close()


def set_tokens(s, k, v):
    """The tokens of the only sequence of s: fp32 k, v [tokens, kv heads, dim]."""
    s.be.cache_append(s.cache, s.layer, s.batch(s.lengths), None, k, v)
    torch.cuda.synchronize()
    s.k, s.v = held(s.kind, k), held(s.kind, v)


@gpu
@pytest.mark.parametrize("new", [3, 200])
@pytest.mark.parametrize("kind,dt", KINDS)
def test_scales_at_the_end_of_fp32(backend, kind, dt, new):
    """Rows of zeros, or rows on keys of zeros, times the largest scales: every token weighs the same, hidden ones nothing."""
    s = Cached(backend, kind, [300], kv_heads=1, dim=64, page=32)
    zeros = torch.zeros((new, 4, 64), dtype=TDT[dt], device="cuda")
    check(s, [new], 4, dt, q=zeros, scale=3e38, window=100)
    set_tokens(s, torch.zeros((300, 1, 64), device="cuda"), normal((300, 1, 64), 3))
    check(s, [new], 4, dt, q=normal((new, 4, 64), 4, dt), scale=3e38, window=100)
    if dt == "bf16":
        check(s, [new], 4, dt, q=normal((new, 4, 64), 4, dt).sign() * 1e38, scale=1e10, window=100)
    s.close()


@gpu
@pytest.mark.parametrize("new", [4, 200])
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("scale", [40.0, 4.1e3, 2.3e6, 1.7e9, 3e20, 1e36])
def test_scores_at_the_end_of_fp32(backend, kind, dt, new, scale):
    """Scores of up to 84 scales in fifteen stairs, 12 scales apart: those on a row's highest stair share it."""
    L, dim = 3000, 64
    s = Cached(backend, kind, [L], kv_heads=2, dim=dim, page=64)
    k, v = normal((L, 2, dim), 3) * 0.25, normal((L, 2, dim), 4)
    k[:, :, 1] = 15.875 if kind == "q8" else 7.0                 # (absmax of its group of 32: d = 1/8, or 1)
    k[:, :, 0] = (torch.arange(L, device="cuda") * 15 // L - 7.0).reshape(-1, 1)
    set_tokens(s, k, v)
    q = torch.zeros((new, 6, dim), dtype=TDT[dt], device="cuda")
    q[:, 0::2, 0], q[:, 1::2, 0], q[:, 4, 0] = 12.0, -12.0, 0.0
    for window in (0, 1700):
        check_each(s, [new], 3, dt, q=q, scale=scale, window=window, exact=kind != "bf16", exact_scores=True)
    s.close()


@gpu
@pytest.mark.parametrize("new", [4, 200])
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_peaks_late_in_a_long_context(backend, kind, dt, dim, new):
    """Scores that climb in fifteen stairs of 12 (2^17 each), or fall, or stand: sums are scaled anew at every stair, in parts and waves of their own.  Of a
    row only one dimension is not 0, and the keys there are multiples of a power of two, so that no kind rounds them, nor do many rows: the bound of
    few holds but for P of bf16."""
    L = 3000
    s = Cached(backend, kind, [L], kv_heads=2, dim=dim, page=64)
    k, v = normal((L, 2, dim), 3) * 0.25, normal((L, 2, dim), 4)
    k[:, :, 1] = 15.875 if kind == "q8" else 7.0                 # (absmax of its group of 32: d = 1/8, or 1)
    k[:, :, 0] = (torch.arange(L, device="cuda") * 15 // L - 7.0).reshape(-1, 1)
    set_tokens(s, k, v)
    q = torch.zeros((new, 6, dim), dtype=TDT[dt], device="cuda")
    q[:, 0::2, 0], q[:, 1::2, 0], q[:, 4, 0] = 12.0, -12.0, 0.0
    q[1, :, 0] = 6.0
    check_each(s, [new], 3, dt, q=q, scale=1.0, exact=kind != "bf16")
    check_each(s, [new], 3, dt, q=q, scale=1.0, exact=kind != "bf16", window=1700)
    check_each(s, [new], 3, dt, q=normal((new, 6, dim), 5, dt), scale=2.0)
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", KINDS)
@pytest.mark.parametrize("below", [10.3, 17.3, 20.3, 23.3, 26.3])
def test_many_small_probabilities_next_to_large_ones(backend, kind, dt, below):
    """A token in every block whose probability is 2^below of the others', and whose value is nothing: y is what the others have, each as exact as its
    own probability is.  Few rows, and many with the prefill mode EXACT."""
    L, dim = 3000, 128
    s = Cached(backend, kind, [L], kv_heads=1, dim=dim, page=64)
    k, v = normal((L, 1, dim), 3), 64.0 + 8.0 * normal((L, 1, dim), 4)
    k[:, :, 0] = 0.0
    k[7::32], v[7::32] = 0.0, 0.0
    k[7::32, :, 0] = 1.0
    set_tokens(s, k, v)
    top = s.k[7, 0, 0].item()
    # y is about 31 tokens of 64 to each large one: 2^(11 - below), in f16 a subnormal number from 2^-14 down, whose half step is 2^-25
    unit = 1.0 if dt == "f16" else 2.0 ** -below
    for new in (2, 100):
        q = torch.zeros((new, 2, dim), dtype=TDT[dt], device="cuda")
        q[:, :, 0] = 4.0
        backend.set_prefill_mode("exact")
        try:
            check_each(s, [new], 2, dt, q=q, scale=below * math.log(2.0) / 4.0 / top, exact=True, unit=unit)
        finally:
            backend.set_prefill_mode("fast")
    s.close()


@gpu
@pytest.mark.parametrize("new", [3, 300])
@pytest.mark.parametrize("power", [110, 60, -60, -90])
def test_values_of_bf16_far_from_one(backend, new, power):
    """Values of 2^power, whose sum over the tokens is within fp32, under scores of 0 in some blocks and 10 in others: less apart than what a maximum may
    lag by, so that probabilities stand far above the first block's."""
    L, dim, kv = 40000, 64, 8
    s = Cached(backend, "bf16", [L], kv_heads=kv, dim=dim, page=32)
    k, v = torch.zeros((L, kv, dim), device="cuda"), (1.0 + 0.5 * normal((L, kv, dim), 4).clamp(-0.9, 0.9)) * 2.0 ** power
    k[:, :, 0] = torch.where(normal((L // 32, kv), 6) < 0.0, 0.0, 10.0).repeat_interleave(32, dim=0)
    set_tokens(s, k, v)
    q = torch.zeros((new, 2 * kv, dim), dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1.0
    check_each(s, [new], 2, "bf16", q=q, scale=1.0, unit=2.0 ** power)
    s.close()


@gpu
def test_batches_that_are_mostly_empty(backend):
    """A prompt and single tokens among as many sequences as a call may have, next to many kv heads: a tile for every sequence and head would be
    a launch of 2^32 threads."""
    B, heads = 65536, 128
    lengths = [0] * B
    lengths[41] = 520
    for i in range(20):
        lengths[3000 * i + 77] = 10 * i + 1
    lengths[B - 1] = 30
    new = [500 if b == 41 else min(n, 1) for b, n in enumerate(lengths)]
    s = Cached(backend, "q4", lengths, kv_heads=heads, dim=64, page=64)
    check_each(s, new, 1, "f16", rows=600)
    s.close()


@gpu
def test_the_largest_call(backend):
    """rows * q_heads / 16 + seqs * kv_heads of 2^24 - 1024 are refused: one unit more than a launch has threads for."""
    import ctypes
    seqs, rows, heads = 7168, 4094, 65536
    assert rows * heads // 16 + seqs == (1 << 24) - 1024
    s = Cached(backend, "q4", [5], kv_heads=1, dim=64, page=32)
    zeros = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")          # sequences without rows
    b = backend.cache_batch(zeros, zeros[1:], zeros[1:].reshape(-1, 1), rows)
    q, y = (torch.full((8, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    status = backend._lib.cybq_attention(backend._ctx, s.cache.handle, 0, b._addr, q.data_ptr(), heads * 64, 1, heads, ctypes.c_float(1.0), 0, y.data_ptr(), None)
    torch.cuda.synchronize()
    assert status == -7 and (y == 7.0).all()
    s.close()


@gpu
@pytest.mark.parametrize("new", [3, 300])
def test_values_at_the_end_of_f16_stay_finite(backend, new):
    """A token in every block with twice the others' probability, less so little that P of f16 is rounded up by all that a rounding can be: on values of
    the largest number y is that number, and not the infinity behind it."""
    L = 700
    s = Cached(backend, "f16", [L], kv_heads=2, dim=64, page=32)
    k, v = torch.zeros((L, 2, 64), device="cuda"), torch.full((L, 2, 64), math.inf, device="cuda")
    k[5::32, :, 0] = 1.0
    v[:, 1] *= -1.0
    set_tokens(s, k, v)
    assert (s.v.abs() == 65504.0).all()
    q = torch.zeros((new, 4, 64), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    y = check_each(s, [new], 2, "f16", q=q, scale=math.log(2.0) - math.log(1.0 + 1.05 * 2.0 ** -11))
    assert (y.abs() >= 65504.0 * (1.0 - 2.0 ** -10)).all()
    s.close()


@gpu
@pytest.mark.parametrize("kind,dt", [("f16", "f16"), ("bf16", "bf16"), ("q8", "f16"), ("q4", "bf16")])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_a_captured_sequence_of_any_number_of_rows(backend, kind, dt, dim):
    """A call of one sequence, recorded for a prompt and replayed with fewer rows, down to one and none, between eager calls: each the bits of a call
    that is made for its rows alone; and the bound of a few rows where they are few, over parts of a long context."""
    L, rows = 5000, 700
    s = Cached(backend, kind, [L], kv_heads=2, dim=dim, page=64)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    starts, lengths = ints([0, rows]), ints([L])
    batch = backend.cache_batch(starts, lengths, s.tables, rows)
    q = normal((rows, 8, dim), 5, dt)
    y = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        backend.attention(s.cache, 0, batch, q, y, stream=torch.cuda.current_stream().cuda_stream)
    for n in (rows, 1, 0, 5, 16, 300, 1, rows):
        starts.copy_(ints([0, n]))
        y.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert (got[n:] == 9.0).all()
        if n:
            alone = check_each(s, [n], 4, dt, q=q[:n].contiguous())
            if n * 4 <= FEW or n == rows:                        # (of rows between, a call made for them may be the other kernel's)
                assert torch.equal(got[:n], alone)
    s.close()
