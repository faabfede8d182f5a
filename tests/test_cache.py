"""The paged cache - cybq_cache_append, cybq_cache_read - against its definition, bit for bit."""
import math
import os
import subprocess

import numpy as np
import pytest

from cyb_amd.backend import Backend, CybqError, load_library

torch = pytest.importorskip("torch")
from tests.cache_lib import TDT, Cached, held, normal, rope_table, turned      # noqa: E402

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


# ---- without a GPU ------------------------------------------------------------------------------------------------

@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_every_byte_of_a_block_has_one_owner(tmp_path):
    """Keys, values and scales of 32 tokens fill a block without gaps or overlaps, and no byte belongs to two tokens."""
    src = tmp_path / "places.hip"
    src.write_text('''
#include "cache_parts.h"
#include <cstdio>
#include <vector>
using namespace cybq;
template <int KIND, int G> int check()
{
    constexpr int dim = 32 * G, data = cache_data_bytes(KIND, dim), half = cache_half_bytes(KIND, dim);
    constexpr int key = KIND == kCacheQ8 ? 8 : KIND == kCacheQ4 ? 4 : 16, value = cache_quantised(KIND) ? 1 : 2;
    for (int what = 0; what < 2; what++) {
        std::vector<int> owner(half, -1);
        auto own = [&](int at, int n, int t) { for (int i = at; i < at + n; i++) { if (i < 0 || i >= half || owner[i] >= 0) return false; owner[i] = t; } return true; };
        for (int t = 0; t < 32; t++) {
            for (int g = 0; g < G; g++) {
                if (!what) for (int q4 = 0; q4 < 4; q4++) { int at = key_place<KIND, G>(t, g, q4); if (at % key || at + key > data || !own(at, key, t)) return 1; }
                if (cache_quantised(KIND) && (scale_place(t, g) % 2 || !own(data + scale_place(t, g), 2, t))) return 2;
            }
            if (what) for (int d = 0; d < dim; d++) {
                if (KIND == kCacheQ4 && (d & 16)) continue;
                int at = value_place<KIND, G>(t, d);
                if (at + value > data || !own(at, value, t)) return 3;
            }
        }
        for (int i = 0; i < half; i++) if (owner[i] < 0) return 4;
    }
    if (half % 16 || cache_block_bytes(KIND, dim) != 2 * half) return 5;
    return 0;
}
template <int KIND> int all() { int r = check<KIND, 2>(); r = r ? r : check<KIND, 3>(); r = r ? r : check<KIND, 4>(); return r ? r : check<KIND, 8>(); }
int main()
{
    int r[4] = {all<kCacheF16>(), all<kCacheBF16>(), all<kCacheQ4>(), all<kCacheQ8>()};
    std::printf("%d %d %d %d\\n", r[0], r[1], r[2], r[3]);
    return r[0] | r[1] | r[2] | r[3];
}
''')
    out = str(tmp_path / "places")
    cc = subprocess.run([HIPCC, "-std=c++17", "--offload-host-only", "-I", os.path.join(ROOT, "cyb_amd", "csrc"), str(src), "-o", out],
                        capture_output=True, text=True)
    assert cc.returncode == 0, cc.stderr[-3000:]
    run = subprocess.run([out], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_null_arguments_are_refused_without_a_device():
    lib = load_library()
    assert lib.cybq_cache_create(None, 8, 1, 1, 128, 64, 1, None) == -1
    assert lib.cybq_cache_free(None, None) == -1
    assert lib.cybq_cache_info(None, None, None, None, None, None, None, None, None, None) == -1
    assert lib.cybq_cache_append(None, None, 0, None, None, 0, 0, None, 0, None, 0, 1, None, 0, 0, 0, None, 1, None) == -1
    assert lib.cybq_cache_read(None, None, 0, None, None, None, 0, None) == -1
    assert lib.cybq_attention(None, None, 0, None, None, 0, 1, 1, 1.0, 0, None, None) == -1


def _dry():
    """A Backend without a device, and a cache and a batch that claim to be on it: the Python checks alone."""
    import ctypes
    from cyb_amd import backend as B
    be = B.Backend.__new__(B.Backend)
    be._lib, be._ctx, be._addr, be.device, be.weights = B.load_library(), ctypes.c_void_p(), 0, 0, {}
    c = B.KVCache.__new__(B.KVCache)
    c._backend, c._h, c._addr, c.kind, c.kv_heads, c.dim, c.layers = be, ctypes.c_void_p(), 0, "q8", 2, 64, 1
    b = B.CacheBatch.__new__(B.CacheBatch)
    b.rows, b._device, b._addr = 3, 0, 0
    return be, c, b


@pytest.mark.parametrize("call,text", [
    ("be.kv_cache('q5', 1, 2, 64, 64, 1)", "unknown cache kind"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), t(3, 2, 64), style='both')", "unknown rope style"),
    ("be.cache_append(c, 0, b, None, t(2, 2, 64), t(3, 2, 64))", "k must be"),
    ("be.cache_append(c, 0, b, None, t(3, 3, 64), t(3, 2, 64))", "k must be"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), t(3, 128))", "v must be"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), t(3, 2, 128)[:, :, ::2])", "must be contiguous"),
    ("be.cache_append(c, 0, b, None, t(3, 4, 64)[:, ::2], t(3, 2, 64))", "must be contiguous"),
    ("be.cache_append(c, 0, b, t(3, 4, 64), t(3, 2, 64), t(3, 2, 64))", "go together"),
    ("be.cache_append(c, 0, b, t(3, 4, 64), t(3, 2, 64), t(3, 2, 64), t(3, 2, 64))", "q_out must be"),
    ("be.cache_append(c, 0, b, t(3, 4, 64), t(3, 2, 64), t(3, 2, 64), t(3, 8, 64)[:, :4])", "q_out must be contiguous"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), t(3, 2, 64).float())", "share one type"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), t(3, 2, 64), rope=t(64, 32, 2))", "rope must be"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64), torch.empty((3, 2, 64), dtype=torch.float16))", "must live on"),
    ("be.cache_append(c, 0, b, None, t(3, 2, 64).int(), t(3, 2, 64).int())", "unsupported dtype"),
    ("be.cache_read(c, 0, b, t(3, 2, 64), t(3, 2, 64).float())", "share one type"),
    ("be.cache_read(c, 0, b, t(3, 4, 64)[:, :2], t(3, 2, 64))", "k must be contiguous"),
    ("be.attention(c, 0, b, t(3, 4, 64), t(3, 4, 64).float())", "share one type"),
    ("be.attention(c, 0, b, t(3, 4, 64), t(2, 4, 64))", "y must be"),
    ("be.attention(c, 0, b, t(3, 4, 96), t(3, 4, 64))", "q must be"),
    ("be.attention(c, 0, b, t(3, 4, 64), t(3, 4, 64))", "already freed"),
    ("be.cache_batch(i(3), i(3), i(3, 4), 1)", "starts must be"),
    ("be.cache_batch(i(4), i(3), i(2, 4), 1)", "starts must be"),
    ("be.cache_batch(i(4).long(), i(3), i(3, 4), 1)", "starts must be int32"),
    ("be.cache_batch(i(4), i(3), i(3, 8)[:, :4], 1)", "tables must be contiguous"),
])
def test_what_the_python_checks_refuse(call, text):
    from torch._subclasses.fake_tensor import FakeTensorMode
    be, c, b = _dry()
    with FakeTensorMode():
        t = lambda *shape: torch.empty(shape, dtype=torch.float16, device="cuda")
        i = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")
        with pytest.raises(CybqError, match=text):
            eval(call, {"be": be, "c": c, "b": b, "t": t, "i": i, "torch": torch})


# ---- refusals of the library -------------------------------------------------------------------------------------------

@gpu
def test_what_cache_create_refuses(backend):
    for args, status in ((("q8", 0, 1, 128, 64, 1), -2), (("q8", 1, 0, 128, 64, 1), -2), (("q8", 1, 1, 80, 64, 1), -2), (("q8", 1, 1, 128, 16, 1), -2),
                         (("q8", 1, 1, 128, 48, 1), -2), (("q8", 1 << 21, 1, 128, 64, 1), -2), (("q8", 1, 4097, 128, 64, 1), -2), (("q8", 1, 1, 128, 2048, 1), -2), (("q8", 1, 1, 128, 64, 0), -2),
                         (("f16", 1 << 20, 4096, 256, 1024, 1 << 30), -2), (("f16", 1 << 10, 64, 256, 1024, 1 << 7), -6)):
        with pytest.raises(CybqError) as e:
            backend.kv_cache(*args)
        assert e.value.status == status, args
    lib = backend._lib
    assert lib.cybq_cache_create(backend._ctx, 5, 1, 1, 128, 64, 1, None) == -1
    c = backend.kv_cache("q4", 3, 5, 96, 128, 7)
    assert (c.kind, c.layers, c.kv_heads, c.dim, c.page, c.pages) == ("q4", 3, 5, 96, 128, 7)
    assert c.page_bytes == 5 * 4 * 2 * (32 * 48 + 192) and c.layer_bytes == 7 * c.page_bytes
    c.free()
    c.free()


@gpu
def test_what_the_calls_refuse(backend):
    import ctypes
    s = Cached(backend, "q8", [5, 40], kv_heads=2, dim=64, page=32)
    lib, h, ctx = backend._lib, s.cache.handle, backend._ctx
    batch = s.batch([1, 2])
    q, y = normal((3, 4, 64), 1, "f16"), torch.full((3, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    kv = normal((3, 2, 64), 2, "f16")
    rope = rope_table(64, 64)

    def attention(cache=h, layer=0, b=batch._addr, x=q.data_ptr(), stride=256, dt=1, heads=4, scale=1.0, window=0, out=y.data_ptr()):
        return lib.cybq_attention(ctx, cache, layer, b, x, stride, dt, heads, ctypes.c_float(scale), window, out, None)

    def append(k=kv.data_ptr(), stride=128, dt=1, r=rope.data_ptr(), positions=64, dims=64, style=0, x=q.data_ptr(), qs=256, heads=4, out=y.data_ptr(), qdt=1):
        return lib.cybq_cache_append(ctx, h, 0, batch._addr, x, qs, heads, k, stride, kv.data_ptr(), 128, dt, r, positions, dims, style, out, qdt, None)

    for kw, status in (({"cache": None}, -1), ({"layer": 1}, -2), ({"layer": -1}, -2), ({"b": None}, -1), ({"x": None}, -1), ({"out": None}, -1),
                       ({"dt": 0}, -1), ({"dt": 9}, -1), ({"heads": 3}, -2), ({"heads": 0}, -2), ({"stride": 255}, -2), ({"stride": 260}, -3),
                       ({"x": q.data_ptr() + 2}, -3), ({"out": y.data_ptr() + 2}, -3), ({"scale": 0.0}, -1), ({"scale": -1.0}, -1),
                       ({"scale": math.inf}, -1), ({"scale": math.nan}, -1), ({"window": -1}, -2)):
        assert attention(**kw) == status, kw
    for kw, status in (({"k": None}, -1), ({"stride": 120}, -2), ({"stride": 132}, -3), ({"dt": 3}, -1), ({"r": rope.data_ptr() + 4}, -3),
                       ({"positions": 63}, -2), ({"dims": 24}, -2), ({"dims": 0}, -2), ({"dims": 80}, -2), ({"style": 2}, -1), ({"out": None}, -1),
                       ({"x": None}, -1), ({"heads": 5}, -2), ({"qs": 250}, -2), ({"qdt": 0}, -1), ({"out": y.data_ptr() + 8}, -3)):
        assert append(**kw) == status, kw
    assert lib.cybq_cache_read(ctx, h, 0, batch._addr, kv.data_ptr(), None, 1, None) == -1
    assert lib.cybq_cache_read(ctx, h, 0, batch._addr, kv.data_ptr(), kv.data_ptr() + 2, 1, None) == -3
    assert lib.cybq_cache_read(ctx, h, 0, batch._addr, kv.data_ptr(), kv.data_ptr(), 7, None) == -1
    for field, value, status in (("seqs", -1, -2), ("seqs", 65537, -2), ("rows", -1, -2), ("rows", (1 << 24) + 1, -2), ("max_new", 0, -2), ("table_pages", 0, -2),
                                 ("table_pages", (1 << 25) + 1, -2), ("starts", None, -1), ("lengths", None, -1), ("tables", None, -1), ("lengths", 4098, -3)):
        b = s.batch([1, 2])
        setattr(b._s, field, value)
        assert attention(b=b._addr) == status, field
    torch.cuda.synchronize()
    assert (y == 7.0).all()                                      # a refused call writes nothing
    for field in ("seqs", "rows"):                               # nothing to do
        b = s.batch([1, 2])
        setattr(b._s, field, 0)
        assert attention(b=b._addr) == 0
    for kind, dt in (("f16", "bf16"), ("bf16", "f16")):
        o = Cached(backend, kind, [3], dim=64)
        with pytest.raises(CybqError) as e:
            backend.attention(o.cache, 0, o.batch([1]), normal((1, 2, 64), 1, dt), torch.empty((1, 2, 64), dtype=TDT[dt], device="cuda"))
        assert e.value.status == -7
        o.close()
    s.close()


# ---- against the definition --------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_rows_are_turned_stored_and_read_back(backend, kind, dim, dt):
    """Three sequences whose new rows begin and end inside blocks and pages, q, k and v slices of one buffer, every byte compared."""
    kv, group, page, lengths, new = 3, 2, 64, [70, 1, 333], [37, 1, 301]
    s = Cached(backend, kind, lengths, kv_heads=kv, dim=dim, page=page, seed=dim)
    rows, heads = sum(new), kv * group
    for style, dims in (("halves", dim), ("pairs", dim // 2), ("halves", 16 if dim == 64 else 32), ("none", 0)):
        qkv = normal((rows + 2, heads + 2 * kv, dim), dim + len(style), dt, std=3.0)
        rope = rope_table(s.tables.shape[1] * page, dims) if dims else None
        batch = s.batch(new, rows=rows + 2)
        q_out = torch.full((rows + 2, heads, dim), 9.0, dtype=torch.bfloat16 if dt == "bf16" else torch.float16, device="cuda")
        backend.cache_append(s.cache, 0, batch, qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], q_out, rope=rope,
                             style="halves" if style == "none" else style)
        k, v = (torch.full((rows + 2, kv, dim), 9.0, device="cuda") for _ in range(2))
        backend.cache_read(s.cache, 0, batch, k, v)
        torch.cuda.synchronize()
        where = [L - n + i for L, n in zip(lengths, new) for i in range(n)]
        x = turned(qkv[:rows], where, rope, style)
        assert torch.equal(q_out[:rows], x[:, :heads].to(q_out.dtype))
        assert torch.equal(k[:rows].double(), held(kind, x[:, heads:heads + kv]))
        assert torch.equal(v[:rows].double(), held(kind, qkv[:rows, heads + kv:]))
        assert (q_out[rows:] == 9.0).all() and (k[rows:] == 9.0).all() and (v[rows:] == 9.0).all()       # rows of no sequence
        # the tokens before the new ones are as they were, in every output type
        for out in TDT:
            ok, ov = (torch.full((sum(lengths), kv, dim), 9.0, dtype=TDT[out], device="cuda") for _ in range(2))
            backend.cache_read(s.cache, 0, s.batch(lengths), ok, ov)
            torch.cuda.synchronize()
            at = row = 0
            for L, n in zip(lengths, new):
                assert torch.equal(ok[at:at + L - n], s.k[at:at + L - n].to(TDT[out])) and torch.equal(ov[at:at + L - n], s.v[at:at + L - n].to(TDT[out]))
                assert torch.equal(ok[at + L - n:at + L], k[row:row + n].to(TDT[out]))
                at += L
                row += n
    s.close()


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8", "q4"])
def test_token_by_token_is_the_same_as_at_once(backend, kind):
    L, kv, dim = 75, 2, 96
    s = Cached(backend, kind, [L], kv_heads=kv, dim=dim, page=32, dt="f32")
    other = Cached(backend, kind, [0], kv_heads=kv, dim=dim, page=32, width=3, spare=3, dt="f32")
    other.tables.copy_(torch.tensor([[2, 0, 1]], dtype=torch.int32))
    for i in range(L):
        b = other.batch([1], lengths=[i + 1])
        backend.cache_append(other.cache, 0, b, None, s.k_in[i:i + 1], s.v_in[i:i + 1])
    k, v = (torch.empty((L, kv, dim), device="cuda") for _ in range(2))
    backend.cache_read(other.cache, 0, other.batch([L], lengths=[L]), k, v)
    torch.cuda.synchronize()
    assert torch.equal(k.double(), s.k) and torch.equal(v.double(), s.v)
    s.close()
    other.close()


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8", "q4"])
def test_what_is_not_finite_or_out_of_range(backend, kind):
    """NaN, infinities, the largest and smallest numbers, signed zeros, groups of zeros, ties of the quantiser."""
    dim, rows = 64, 12
    x = normal((rows, 1, dim), 3)
    x[0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 3.4e38], device="cuda")
    x[1] = math.nan
    x[2] = -math.inf
    x[3] = 0.0
    x[4] = -0.0
    x[5] = 1e-45
    x[6] *= 1e-7
    x[7] *= 1e30
    x[8, 0, :32] = torch.arange(32, device="cuda") * 0.5 - 7.5                    # absmax 8 (7.5): halves of the step
    x[8, 0, 32:] = torch.arange(32, device="cuda") * 8.0 - 127.0
    x[9] = 65520.0
    x[10] = 57344.0
    x[11, 0, 0] = 6.1e-5
    s = Cached(backend, kind, [0], kv_heads=1, dim=dim, page=32, spare=1)
    s.tables[0, 0] = 0
    b = s.batch([rows], lengths=[rows])
    backend.cache_append(s.cache, 0, b, None, x, -x)
    k, v = (torch.empty((rows, 1, dim), device="cuda") for _ in range(2))
    backend.cache_read(s.cache, 0, b, k, v)
    torch.cuda.synchronize()
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    assert torch.equal(k.double(), held(kind, x)) and torch.equal(v.double(), held(kind, -x))
    half = torch.empty((rows, 1, dim), dtype=torch.float16, device="cuda")
    if kind != "bf16":
        backend.cache_read(s.cache, 0, b, half, half.clone())
        torch.cuda.synchronize()
        assert torch.isfinite(half).all()
    s.close()


@gpu
def test_tokens_without_a_place(backend):
    """Pages that are none, positions below zero and behind the table: not stored, read as zeros, q zeros where there is no position."""
    kv, dim, page = 2, 64, 32
    s = Cached(backend, "q8", [96, 5, 40], kv_heads=kv, dim=dim, page=page, width=3)
    s.tables[0, 1] = -1
    s.tables[2, 1] = s.cache.pages
    before = [torch.empty((s.cache.pages * page, kv, dim), device="cuda") for _ in range(2)]
    every = backend.cache_batch(torch.tensor([0, s.cache.pages * page], dtype=torch.int32, device="cuda"),
                                torch.tensor([s.cache.pages * page], dtype=torch.int32, device="cuda"),
                                torch.arange(s.cache.pages, dtype=torch.int32, device="cuda").reshape(1, -1), s.cache.pages * page)
    backend.cache_read(s.cache, 0, every, *before)
    # 96 rows with a hole; nine rows of a sequence of five tokens; 40 rows up to position 109 of a table of 96
    new, lengths = [96, 9, 40], [96, 5, 110]
    rows = sum(new)
    x = normal((rows, 2 * kv, dim), 5, "f16")
    q_out = torch.full((rows, kv, dim), 9.0, dtype=torch.float16, device="cuda")
    b = s.batch(new, lengths=lengths)
    backend.cache_append(s.cache, 0, b, x[:, :kv], x[:, :kv], x[:, kv:], q_out, rope=rope_table(96, dim))
    k, v = (torch.full((rows, kv, dim), 9.0, device="cuda") for _ in range(2))
    backend.cache_read(s.cache, 0, b, k, v)
    torch.cuda.synchronize()
    where = np.array([L - n + i for L, n in zip(lengths, new) for i in range(n)])
    seq = np.repeat(np.arange(3), new)
    placed = (where >= 0) & (where < 96)
    table = s.tables.cpu().numpy()
    paged = placed & (np.array([0 <= table[b, p // page] < s.cache.pages if ok else False for b, p, ok in zip(seq, where, placed)]))
    t, paged = turned(x[:, :kv], where, rope_table(96, dim), "halves"), torch.from_numpy(paged).cuda().reshape(-1, 1, 1)
    assert torch.equal(q_out, torch.where(torch.from_numpy(placed).cuda().reshape(-1, 1, 1), t.half(), 0.0))
    assert torch.equal(k.double(), torch.where(paged, held("q8", t), 0.0)) and torch.equal(v.double(), torch.where(paged, held("q8", x[:, kv:]), 0.0))
    # nothing else in the cache moved
    after = [torch.empty_like(t) for t in before]
    backend.cache_read(s.cache, 0, every, *after)
    torch.cuda.synchronize()
    written = {int(table[b, p // page]) * page + p % page for b, p, ok in zip(seq, where, paged.flatten().tolist()) if ok}
    rest = torch.tensor([i for i in range(s.cache.pages * page) if i not in written], device="cuda")
    assert torch.equal(before[0][rest], after[0][rest]) and torch.equal(before[1][rest], after[1][rest])
    s.close()


@gpu
def test_many_sequences_layers_and_copied_pages(backend):
    """More sequences than a wave has lanes, some without rows; another layer is left alone; a page's bytes mean the same elsewhere."""
    kv, dim, page, B = 1, 64, 32, 150
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 90, B).tolist()
    lengths[70] = 0
    s = Cached(backend, "q4", lengths, kv_heads=kv, dim=dim, page=page, layers=3, layer=1, width=3)
    new = [min(L, int(n)) for L, n in zip(lengths, rng.integers(0, 50, B))]
    rows = sum(new)
    at = np.concatenate([[0], np.cumsum(lengths)])
    tokens = torch.tensor([at[b] + L - n + i for b, (L, n) in enumerate(zip(lengths, new)) for i in range(n)], device="cuda")
    k, v = (torch.empty((rows, kv, dim), device="cuda") for _ in range(2))
    backend.cache_read(s.cache, 1, s.batch(new), k, v)
    torch.cuda.synchronize()
    assert torch.equal(k.double(), s.k[tokens]) and torch.equal(v.double(), s.v[tokens])
    for layer in (0, 2):
        backend.cache_read(s.cache, layer, s.batch(new), k, v)
        torch.cuda.synchronize()
        assert (k == 0).all() and (v == 0).all()
    # layer 1 to layer 2, pages turned round
    import ctypes
    hip, c = backend._lib, s.cache                               # (the runtime that the library is linked with)
    for p in range(c.pages):
        rc = hip.hipMemcpy(ctypes.c_void_p(c.memory + 2 * c.layer_bytes + (c.pages - 1 - p) * c.page_bytes),
                           ctypes.c_void_p(c.memory + c.layer_bytes + p * c.page_bytes), ctypes.c_size_t(c.page_bytes), 3)
        assert rc == 0
    s.tables.copy_(torch.where(s.tables >= 0, c.pages - 1 - s.tables, -1))
    backend.cache_read(s.cache, 2, s.batch(new), k, v)
    torch.cuda.synchronize()
    assert torch.equal(k.double(), s.k[tokens]) and torch.equal(v.double(), s.v[tokens])
    s.close()


@gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [3, 40])
def test_queries_that_do_not_turn_are_as_they_were(backend, dt, new):
    """Infinities, NaN and signed zeros in dimensions that do not turn - all of them without angles, those behind rope_dims with - reach q_out as
    they are, and none of them another dimension."""
    kv, group, dim, page = 2, 3, 64, 32
    s = Cached(backend, "q8", [50], kv_heads=kv, dim=dim, page=page)
    for style, dims in (("none", 0), ("halves", 32), ("pairs", 16)):
        x = normal((new, kv * group, dim), 7, dt)
        for row in range(new):                                   # (every pair of neighbours and of halves meets each of them somewhere)
            for head in range(kv * group):
                at = dims + (5 * row + 11 * head) % (dim - dims)
                x[row, head, at] = (math.inf, -math.inf, math.nan)[(row + head) % 3]
                x[row, head, dims + (at - dims + 3) % (dim - dims)] = -0.0
        rope = rope_table(s.tables.shape[1] * page, dims) if dims else None
        k = normal((new, kv, dim), 8, dt)
        want = turned(x, list(range(50 - new, 50)), rope, style)
        for qdt in (torch.float16, torch.bfloat16):
            q_out = torch.full((new, kv * group, dim), 9.0, dtype=qdt, device="cuda")
            backend.cache_append(s.cache, 0, s.batch([new]), x, k, k, q_out, rope=rope, style="halves" if style == "none" else style)
            torch.cuda.synchronize()
            bad = torch.isnan(x)
            assert torch.equal(torch.isnan(q_out), bad)
            assert torch.equal(q_out.view(torch.int16)[~bad], want.to(qdt).view(torch.int16)[~bad])
    s.close()


def test_a_backend_that_closes_frees_its_caches():
    """cybq_cache_free for every cache that is still there, before cybq_destroy; not again afterwards, nor for one that was freed."""
    import ctypes
    import weakref
    from cyb_amd import backend as B

    class Library:
        def __init__(self):
            self.calls, self.made = [], 0

        def cybq_cache_create(self, ctx, kind, layers, heads, dim, page, pages, out):
            self.made += 1
            ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = 4096 * self.made
            return 0

        def cybq_cache_info(self, h, kind, *rest):
            kind.value = 8
            return 0

        def cybq_cache_free(self, ctx, h):
            assert ctx.value == 64
            self.calls.append(h.value)
            return 0

        def cybq_destroy(self, ctx):
            self.calls.append("destroy")

    be = B.Backend.__new__(B.Backend)
    be._lib, be._ctx, be._addr, be.device, be.weights, be._caches = Library(), ctypes.c_void_p(64), 64, 0, {}, weakref.WeakSet()
    first, second, third = (be.kv_cache("q8", 1, 2, 64, 64, 1) for _ in range(3))
    second.free()
    be.close()
    assert be._lib.calls[0] == 8192 and sorted(be._lib.calls[1:3]) == [4096, 12288] and be._lib.calls[3:] == ["destroy"]
    for c in (first, second, third):
        c.free()
        with pytest.raises(CybqError, match="already freed"):
            c.handle
    assert len(be._lib.calls) == 4


@gpu
def test_a_closed_backend_holds_no_cache():
    be = Backend(0)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    cache = be.kv_cache("f16", 2, 8, 128, 64, 4096)              # 2 GiB
    assert torch.cuda.mem_get_info()[0] < before - (1 << 30)
    be.close()
    assert torch.cuda.mem_get_info()[0] >= before
    cache.free()
