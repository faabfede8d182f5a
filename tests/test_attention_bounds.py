"""Attention over the paged cache in calls whose sizes say little about their rows, with scales of any size.  Against float64; the bound of an element is that of
test_attention.py."""
import pytest

torch = pytest.importorskip("torch")
from tests.cache_lib import TDT, Cached, held, normal      # noqa: E402
from tests.test_attention import FEW, KINDS, bound, check  # noqa: E402

gpu = pytest.mark.gpu


def check_each(s, new, group, dt, window=0, scale=None, rows=None, max_new=None, q=None, seed=9, exact=False, unit=1.0):
    """As `check`, each sequence against the bound of its own number of rows (exact: of few), values counted in `unit`.  Scores of any size: what
    the exponent's argument and the factors that scale sums anew lose, at most 4 U of the largest score, is counted as four dimensions more."""
    rows = sum(new) if rows is None else rows
    q = normal((rows, s.kv_heads * group, s.dim), seed, dt) if q is None else q
    y = torch.full(q.shape, 9.0, dtype=TDT[dt], device="cuda")
    s.be.attention(s.cache, s.layer, s.batch(new, rows=rows, max_new=max_new), q, y, scale=scale, window=window)
    torch.cuda.synchronize()
    used = sum(new)
    ref, size, dots = s.expected(q[:used], new, scale, window)
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
