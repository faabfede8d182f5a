"""Mixture of experts - cybq_route, cybq_matmul_experts, cybq_matmul_experts_sum - against their definitions in float64.

Bars of the products, relative L2 per row of y: sums are fp32 over exact operands.  The matrix pipe cuts each of the 33
addends of a group's sum at 2^-24 of the largest, which with biased operands is up to 144 / 3.2 of a typical product
(Q8: 256 / 56): sqrt(33 G) 2^-24 * 3 * 144 s against sqrt(32 G) * 3.2 s for the row, below 1e-5 whatever G is.  TIGHT
doubles that; SwiGLU multiplies two such numbers and has a slope of at most 1.1 in front of one: three times TIGHT.
Outputs of 16 bits add half a step each."""
import ctypes

import numpy as np
import pytest

from cyb_amd import formats
from cyb_amd.backend import Backend, CybqError, QWeight, load_library

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TIGHT = 2e-5
TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# ---- the router --------------------------------------------------------------------------------------------------

def _route_ref(z, k, score="softmax", bias=None, groups=1, top_groups=1, group_best=1, renorm=True, scale=1.0):
    """One row at a time, sorting (-c, index) pairs."""
    T, E = z.shape
    ids, weights = np.zeros((T, k), np.int32), np.zeros((T, k))
    size = E // groups
    for t in range(T):
        row = [float("-inf") if v != v else float(v) for v in z[t].tolist()]
        if score == "sigmoid":
            s = [0.0 if v == float("-inf") else 1.0 / (1.0 + np.exp(-v)) for v in row]
        else:
            top = max(row)
            if top == float("-inf"):
                s = [0.0] * E
            elif top == float("inf"):
                s = [1.0 if v == top else 0.0 for v in row]
            else:
                s = [float(np.exp(v - top)) for v in row]
            total = sum(s)
            s = [v / total if total else 0.0 for v in s]
        if bias is None:
            c, rank = s, row
        else:
            c = rank = [float("-inf") if b != b else v + float(b) for v, b in zip(s, bias.tolist())]
        allowed = range(E)
        if groups > 1:
            best = []
            for g in range(groups):
                v = sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_best])
                best.append((-v if v == v else float("inf"), g))
            allowed = [e for _, g in sorted(best)[:top_groups] for e in range(g * size, (g + 1) * size)]
        chosen = [e for _, e in sorted((-rank[e], e) for e in allowed)[:k]]
        w = [s[e] for e in chosen]
        if renorm:
            total = sum(w)
            w = [v / total if total else 0.0 for v in w]
        ids[t], weights[t] = chosen, [v * np.float64(np.float32(scale)) for v in w]
    return ids, weights


def _route(be, z, k, stream=0, **kw):
    T = z.shape[0]
    ids = torch.full((T + 1, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T + 1, k), -7.0, dtype=torch.float32, device="cuda")
    if "bias" in kw and kw["bias"] is not None:
        kw = dict(kw, bias=torch.from_numpy(np.asarray(kw["bias"], dtype=np.float32)).cuda())
    if "renorm" in kw:
        kw["renormalise"] = kw.pop("renorm")
    be.route(z, ids[:T], w[:T], stream=stream, **kw)
    torch.cuda.synchronize()
    assert (ids[T] == -7).all() and (w[T] == -7).all()               # the row behind the last token
    return ids[:T].cpu().numpy(), w[:T].cpu().numpy()


def _check_route(be, z, k, **kw):
    ids, w = _route(be, z, k, **kw)
    rid, rw = _route_ref(z.double().cpu().numpy(), k, **kw)
    assert np.array_equal(ids, rid)
    assert not np.isnan(w).any()
    np.testing.assert_allclose(w, rw, rtol=2.0 ** -24 + 1e-13, atol=2.0 ** -149)


@gpu
@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (8, 2), (63, 5), (64, 8), (65, 64), (128, 8), (160, 6), (256, 8), (1000, 10), (1024, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_sizes(backend, E, k, score):
    rng = np.random.default_rng(E * 100 + k)
    for dt in ("f32", "f16", "bf16"):
        z = torch.from_numpy(rng.standard_normal((33, E)).astype(np.float32) * 2).cuda().to(TDT[dt])       # (16 bits: many ties)
        _check_route(backend, z, k, score=score)
        _check_route(backend, z, k, score=score, bias=rng.standard_normal(E).astype(np.float32) * 0.1, renorm=False, scale=2.5)


@gpu
@pytest.mark.parametrize("E,groups,top_groups,k", [(256, 8, 4, 8), (160, 8, 3, 6), (64, 64, 8, 8), (64, 2, 1, 32), (1024, 64, 4, 64), (60, 4, 1, 15), (9, 3, 2, 1)])
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(backend, E, groups, top_groups, k, group_best, score):
    rng = np.random.default_rng(E + groups)
    z = torch.from_numpy(rng.standard_normal((40, E)).astype(np.float32)).cuda()
    for bias in (None, rng.standard_normal(E).astype(np.float32) * 0.2):
        _check_route(backend, z, k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best)


@gpu
def test_route_ties_and_values_at_the_ends(backend):
    inf, nan, E = float("inf"), float("nan"), 72
    rows = [np.zeros(E), np.full(E, -inf), np.full(E, nan), np.full(E, inf), np.full(E, 200.0), np.full(E, -3.4e38)]
    a = np.full(E, -inf)
    a[[70, 3]] = 1.0                              # two experts stand, the rest have no score
    b = np.arange(E) % 3.0                        # ties in runs
    c = np.where(np.arange(E) == 40, inf, 1.0)
    d = np.where(np.arange(E) % 2, nan, 0.5)
    e = np.linspace(-90, 90, E)                   # sigmoids that fp32 would round to 0 and 1
    z = torch.from_numpy(np.stack(rows + [a, b, c, d, e]).astype(np.float32)).cuda()
    bias = np.zeros(E, np.float32)
    bias[5], bias[6], bias[7] = -inf, nan, 0.25
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            _check_route(backend, z, 6, score=score, renorm=renorm)
            _check_route(backend, z, 6, score=score, renorm=renorm, bias=bias)
            _check_route(backend, z, 6, score=score, renorm=renorm, groups=9, top_groups=2, group_best=2)
            _check_route(backend, z, 6, score=score, renorm=renorm, bias=bias, groups=9, top_groups=2, group_best=2)


@gpu
def test_route_chooses_where_fp32_could_not(backend):
    """Scores whose sums with the bias differ below fp32's step: the choice is the definition's."""
    E, T = 128, 64
    rng = np.random.default_rng(9)
    z = torch.from_numpy((rng.standard_normal((T, E)) * 1e-8).astype(np.float32)).cuda()
    _check_route(backend, z, 8, score="sigmoid", bias=np.full(E, 3.0, np.float32))
    _check_route(backend, z, 8, score="softmax", bias=np.full(E, 3.0, np.float32))


@gpu
@pytest.mark.parametrize("T", [0, 1, 255, 256, 257, 3001])
def test_route_token_counts(backend, T):
    rng = np.random.default_rng(T)
    z = torch.from_numpy(rng.standard_normal((T, 96)).astype(np.float32)).cuda()
    _check_route(backend, z, 4, score="sigmoid", bias=rng.standard_normal(96).astype(np.float32), groups=6, top_groups=3, group_best=2)


# ---- the products ------------------------------------------------------------------------------------------------

def _stack(be, bits, E, n, K, seed, scale=0.01):
    """A stack of experts and its float64 values [E, n, K]."""
    rng = np.random.default_rng(seed)
    q = rng.integers(-8 if bits == 4 else -127, 8 if bits == 4 else 128, size=(E * n, K), dtype=np.int8)
    s = ((0.5 + rng.random((E * n, K // 32), dtype=np.float32)) * (scale if bits == 4 else scale / 16)).astype(np.float16)
    wd = torch.from_numpy(s).cuda().double().repeat_interleave(32, dim=1) * torch.from_numpy(q).cuda()
    return be.upload_quantized(q, s.view(np.uint16), bits), wd.reshape(E, n, K)


def _rows(shape, dt, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(generator=g).to(TDT[dt])


def _ids(T, k, E, seed, how="spread"):
    rng = np.random.default_rng(seed)
    if how == "one":
        a = np.full((T, k), E - 1)
    elif how == "few":
        a = rng.integers(0, min(E, 2), size=(T, k))
    elif how == "none":
        a = np.full((T, k), -1)
    else:
        a = rng.integers(0, E, size=(T, k))
        if how == "padded":
            a[rng.random((T, k)) < 0.3] = -1
            a[T - T // 3:] = rng.choice([-1, E, E + 7, 2 ** 31 - 1, -2 ** 31], size=(T // 3, k))
    return torch.from_numpy(a.astype(np.int32)).cuda()


def _products(x, xdiv, wd, ids):
    """float64 [P, n], zeros for pairs without an expert."""
    flat = ids.reshape(-1).long()
    out = torch.zeros((flat.numel(), wd.shape[1]), dtype=torch.float64, device="cuda")
    for e in range(wd.shape[0]):
        p = torch.nonzero(flat == e).reshape(-1)
        if p.numel():
            out[p] = x.double()[p // xdiv] @ wd[e].T.contiguous()
    return out


def _close(got, ref, bar, what=""):
    err = (got.double() - ref).norm(dim=1) / ref.norm(dim=1).clamp_min(1e-300)
    assert not torch.isnan(got).any(), what
    assert err.max().item() < bar, (what, err.max().item(), err.argmax().item())


def _check_up(be, bits, E, n, K, T, k, xdt, ydt, how="spread", swiglu=False, seed=0, stream=0):
    ids = _ids(T, k, E, seed + 1, how)
    x = _rows((T, K), xdt, seed + 2)
    w, wd = _stack(be, bits, E, n, K, seed + 3)
    ref = _products(x, k, wd, ids)
    if swiglu:
        u, ud = _stack(be, bits, E, n, K, seed + 4)
        w = be.fuse_pairs(w, u)
        ref = ref * torch.sigmoid(ref) * _products(x, k, ud, ids)
    y = torch.full((T * k + 1, n), float("nan"), dtype=TDT[ydt], device="cuda")
    be.matmul_experts(w, E, x, ids, y[:T * k], "swiglu" if swiglu else "none", stream=stream)
    torch.cuda.synchronize()
    has = ((ids >= 0) & (ids < E)).reshape(-1)
    assert torch.isnan(y[T * k]).all() and torch.isnan(y[:-1][~has]).all()          # rows without an expert stay as they were
    if has.any():
        _close(y[:-1][has], ref[has], (3 if swiglu else 1) * TIGHT + HALF_STEP[ydt], (bits, E, n, K, T, k, xdt, ydt, how, swiglu))
    w.free()


def _check_down(be, bits, E, n, K, T, k, xdt, ydt, how="spread", residual=True, seed=0, alias=False):
    ids = _ids(T, k, E, seed + 1, how)
    x = _rows((T * k, K), xdt, seed + 2)
    w, wd = _stack(be, bits, E, n, K, seed + 3)
    g = _rows((T, k), "f32", seed + 5)
    r = _rows((T, n), ydt, seed + 6) if residual else None
    z = _products(x, 1, wd, ids) * g.double().reshape(-1, 1)
    ref = z.reshape(T, k, n).sum(dim=1) + (r.double() if residual else 0.0)
    # every pair's product has an error of its own: relative to their root sum of squares
    size = (z.reshape(T, k, n) ** 2).sum(dim=(1, 2)).sqrt() + (r.double().norm(dim=1) if residual else 0.0)
    y = torch.full((T + 1, n), float("nan"), dtype=TDT[ydt], device="cuda")
    if alias:
        y[:T] = r
        r = y[:T]
    be.matmul_experts_sum(w, E, x, ids, g, y[:T], r)
    torch.cuda.synchronize()
    assert torch.isnan(y[T]).all() and not torch.isnan(y[:T]).any()
    err = (y[:T].double() - ref).norm(dim=1)
    bar = TIGHT * size + HALF_STEP[ydt] * ref.norm(dim=1) + 1e-300
    assert (err <= bar).all(), (bits, E, n, K, T, k, xdt, ydt, how, (err / bar).max().item())
    w.free()


@gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("xdt", ["f16", "bf16", "f32"])
# K that ends inside a tile, one group, several tiles per wave; one strip, odd strips; one token to a few rows per expert
@pytest.mark.parametrize("E,n,K,T,k", [(1, 16, 32, 1, 1), (4, 48, 96, 1, 2), (16, 32, 2048, 1, 8), (16, 80, 1312, 3, 4), (60, 32, 160, 7, 6), (8, 64, 4224, 16, 2),
                                       (3, 16, 128, 64, 8), (8, 96, 256, 65, 8), (200, 16, 64, 70, 3), (5, 16, 32, 4, 64), (4, 48, 4256, 2, 3), (40, 32, 1056, 16, 8)])
def test_few_rows(backend, bits, xdt, E, n, K, T, k):
    for swiglu in (False, True):
        _check_up(backend, bits, E, n, K, T, k, xdt, "f32", swiglu=swiglu, seed=K)
    _check_down(backend, bits, E, n, K, T, k, xdt, "f32", seed=K + 1)


@gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("xdt", ["f16", "bf16", "f32"])
# 16 rows and more for every expert, in tiles of 1 to 8 blocks of 16 rows; K of one group, of a part of a tile behind whole ones
@pytest.mark.parametrize("E,n,K,T,k", [(1, 16, 32, 16, 1), (2, 48, 160, 16, 2), (4, 272, 2048, 64, 2), (4, 528, 480, 100, 4), (3, 64, 1024, 129, 3), (1, 32, 256, 257, 1),
                                       (16, 112, 608, 300, 4), (5, 256, 2336, 333, 2)])
def test_many_rows(backend, bits, xdt, E, n, K, T, k):
    for swiglu in (False, True):
        _check_up(backend, bits, E, n, K, T, k, xdt, "f32", swiglu=swiglu, seed=K)
    _check_down(backend, bits, E, n, K, T, k, xdt, "f32", seed=K + 1)


@gpu
@pytest.mark.parametrize("how", ["one", "few", "none", "padded"])
@pytest.mark.parametrize("T,k", [(1, 4), (9, 8), (64, 8), (65, 8), (400, 4)])
def test_uneven_and_missing_experts(backend, how, T, k):
    """All pairs with one expert, the same expert twice for a token, ids that are no expert, none at all."""
    for bits, xdt, ydt in ((4, "f16", "f16"), (8, "bf16", "bf16"), (4, "f32", "f32")):
        _check_up(backend, bits, 24, 64, 352, T, k, xdt, ydt, how, swiglu=True, seed=T)
        _check_down(backend, bits, 24, 64, 352, T, k, xdt, ydt, how, seed=T + 1)
        _check_down(backend, bits, 24, 64, 352, T, k, xdt, ydt, how, residual=False, seed=T + 2)


@gpu
@pytest.mark.parametrize("T", [2, 200])
def test_residual_in_place_and_outputs_of_16_bits(backend, T):
    for xdt in ("f16", "bf16"):
        for ydt in ("f16", "bf16", "f32"):
            _check_down(backend, 4, 8, 96, 512, T, 2, xdt, ydt, alias=True, seed=7)
            _check_up(backend, 4, 8, 96, 512, T, 2, xdt, ydt, seed=8)


@gpu
def test_no_tokens(backend):
    w, _ = _stack(backend, 4, 4, 32, 64, 0)
    x, ids, y = torch.empty((0, 64), device="cuda"), torch.empty((0, 2), dtype=torch.int32, device="cuda"), torch.empty((0, 32), device="cuda")
    backend.matmul_experts(w, 4, x, ids, y)
    backend.matmul_experts_sum(w, 4, x, ids, torch.empty((0, 2), device="cuda"), y)
    w.free()


@gpu
def test_more_tokens_than_a_round(backend):
    """Rounds of 2^20 pairs and of 65535 tokens."""
    _check_up(backend, 4, 4, 16, 32, 16384 + 5, 64, "bf16", "bf16", "padded", seed=1)
    _check_down(backend, 4, 4, 16, 32, 65535 + 70, 2, "f16", "f16", "padded", seed=2)


@gpu
def test_a_token_whose_sums_do_not_fit_the_scratch(backend):
    """64 experts of 2^20 outputs: 256 MiB of fp32 sums per token."""
    n, k, T = 1 << 20, 64, 2
    q = torch.randint(0, 256, (n * 16,), dtype=torch.uint8, device="cuda")
    w = backend.weight_from_device(4, n, 32, q, torch.full((n,), 0x1C00, dtype=torch.int16, device="cuda"))          # scales 2^-8
    x, g = _rows((T * k, 32), "f16", 1), _rows((T, k), "f32", 2)
    y = torch.empty((T, n), device="cuda")
    backend.matmul_experts_sum(w, 1, x, torch.zeros((T, k), dtype=torch.int32, device="cuda"), g, y)
    torch.cuda.synchronize()
    b = q.reshape(n, 16).short()
    v = torch.stack([b & 15, b >> 4], dim=2).reshape(n, 32).double()
    wd = torch.where(v >= 8, v - 16, v) / 256
    mixed = (x.double().reshape(T, k, 32) * g.double()[:, :, None]).sum(dim=1)
    size = (x.double().reshape(T, k, 32).norm(dim=2) * g.double().abs()).norm(dim=1) / mixed.norm(dim=1)
    _close(y, mixed @ wd.T.contiguous(), TIGHT * size.max().item())
    w.free()


@gpu
def test_row_tiles_beyond_one_grid(backend):
    """2^20 pairs on wide experts: more row tiles by strips than a grid has threads for; nearly all pairs have no expert."""
    E, n, K, T, k = 2, 1 << 16, 32, 65535, 16
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("y alone is 137 GB")
    gate, gd = _stack(backend, 4, E, n, K, 1)
    up, ud = _stack(backend, 4, E, n, K, 2)
    w = backend.fuse_pairs(gate, up)
    x = _rows((T, K), "bf16", 3)
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    at = torch.tensor([0, 1, 40000, T - 1], device="cuda")
    ids[at, torch.tensor([0, 15, 7, 15], device="cuda")] = torch.tensor([1, 0, 1, 0], dtype=torch.int32, device="cuda")
    pairs = (ids.reshape(-1) >= 0).nonzero().reshape(-1)
    y = torch.empty((T * k, n), dtype=torch.bfloat16, device="cuda")
    y[pairs[-1] - 1] = 7.0
    backend.matmul_experts(w, E, x, ids, y, "swiglu")
    torch.cuda.synchronize()
    some, e = x[at].contiguous(), ids.reshape(-1)[pairs].reshape(-1, 1).contiguous()
    ref = _products(some, 1, gd, e)
    ref = ref * torch.sigmoid(ref) * _products(some, 1, ud, e)
    _close(y[pairs], ref, 3 * TIGHT + HALF_STEP["bf16"])
    assert (y[pairs[-1] - 1] == 7.0).all()
    del y
    torch.cuda.empty_cache()
    w.free()
    q = torch.zeros(((1 << 26) + 16) * 16, dtype=torch.uint8, device="cuda")
    s = torch.zeros((1 << 26) + 16, dtype=torch.int16, device="cuda")
    w = backend.weight_from_device(4, (1 << 26) + 16, K, q, s)
    with pytest.raises(Exception, match="2\\^26 rows"):
        backend.matmul_experts(w, 1, x[:1], ids[:1, :1].contiguous(), torch.empty((1, (1 << 26) + 16), dtype=torch.float16, device="cuda"))
    torch.cuda.synchronize()
    w.free()


@gpu
def test_rows_that_are_not_finite_stay_among_themselves(backend):
    E, n, K, k = 4, 64, 352, 2
    w, wd = _stack(backend, 4, E, n, K, 3)
    for T in (5, 200):
        for dt in ("f16", "bf16", "f32"):
            x = _rows((T, K), dt, 4)
            ids = _ids(T, k, E, 5)
            x[1, 7], x[3, K - 1] = float("inf"), float("nan")
            bad = torch.zeros(T, dtype=torch.bool, device="cuda")
            bad[[1, 3]] = True
            rows = bad.repeat_interleave(k)
            ref = _products(torch.where(bad[:, None], 0, x), k, wd, ids)
            for ydt in ("f32", "bf16"):                               # (many rows and bf16: rounded operands)
                y = torch.empty((T * k, n), device="cuda", dtype=TDT[ydt])
                backend.matmul_experts(w, E, x, ids, y)
                torch.cuda.synchronize()
                assert not torch.isfinite(y[rows]).any()
                _close(y[~rows], ref[~rows], TIGHT + HALF_STEP[ydt], (T, dt, ydt))
    w.free()


@gpu
def test_rows_of_any_size_and_wide_scales(backend):
    """bf16 and fp32 rows of 1e-30 and 1e30, scales whose products with q leave f16's range."""
    E, n, K, k = 3, 32, 256, 1
    for scale in (0.01, 3.0e4):
        w, wd = _stack(backend, 4, E, n, K, 6, scale)
        for T in (2, 90):
            for dt in ("bf16", "f32"):
                size = torch.tensor([1e-30, 1e30 if scale < 1 else 1e25, 1.0], device="cuda").repeat(T)[:T, None]
                x = (_rows((T, K), "f32", 8) * size).to(TDT[dt])
                ids = _ids(T, k, E, 9)
                y = torch.empty((T * k, n), device="cuda")
                backend.matmul_experts(w, E, x, ids, y)
                torch.cuda.synchronize()
                _close(y, _products(x, k, wd, ids), TIGHT, (scale, T, dt))
        w.free()


@gpu
def test_fp32_rows_keep_their_bits(backend):
    """fp32 rows are not rounded on the way in: an error of one bf16 or f16 step of x would show at 4e-3 / 5e-4."""
    E, n, K = 2, 16, 128
    w, wd = _stack(backend, 8, E, n, K, 1)
    x = _rows((4, K), "f32", 2)
    x = torch.cat([x, -x * (1 + 2.0 ** -20)], dim=0)
    ids = torch.zeros((8, 1), dtype=torch.int32, device="cuda")
    y = torch.empty((8, n), device="cuda")
    backend.matmul_experts(w, E, x, ids, y)
    torch.cuda.synchronize()
    _close(y, _products(x, 1, wd, ids), 2e-6)
    w.free()


@pytest.fixture
def tuned(backend):
    yield backend.set_experts_tuning
    backend.set_experts_tuning()


@gpu
@pytest.mark.parametrize("cols", [1, 2, 4, 8])
@pytest.mark.parametrize("T", [1, 2, 9, 40, 150])
def test_few_rows_whatever_the_waves_do(backend, tuned, cols, T):
    """One row and up to 8, 16, 32, 64 at a time and the rest, K shorter than the waves that share it out, strips that no workgroup divides."""
    tuned(cols, 1 << 20, 2)
    for bits in (4, 8):
        for xdt in ("f16", "bf16", "f32"):
            for n, K in ((144, 1312), (16, 96), (208, 32)):
                _check_up(backend, bits, 3, n, K, T, 2, xdt, "f32", "padded", seed=T)
            _check_up(backend, bits, 3, 112, 864, T, 1, xdt, xdt, "few", swiglu=True, seed=T)
            _check_down(backend, bits, 3, 144, 1312, T, 2, xdt, "f32", seed=T)


@gpu
@pytest.mark.parametrize("T", [1, 5, 33])
def test_the_way_back_token_by_token(backend, tuned, T):
    tuned(0, 0, 1)
    for bits in (4, 8):
        for xdt in ("f16", "bf16", "f32"):
            for E, n, K, k, how in ((3, 16, 32, 1, "spread"), (9, 144, 1312, 3, "padded"), (5, 48, 4128, 7, "few"), (4, 32, 160, 64, "padded")):
                _check_down(backend, bits, E, n, K, T, k, xdt, "f32" if K > 100 else xdt, how, seed=K)


@gpu
@pytest.mark.parametrize("mode", ["fast", "exact"])
@pytest.mark.parametrize("T", [1, 17, 40, 70, 100, 113, 128, 300])
def test_many_rows_whatever_the_mode(backend, tuned, mode, T):
    """All row blocks of a tile; K of whole tiles, of 1, 2 and 3 groups behind them or alone.  With a y of bf16 FAST mode rounds the operands."""
    tuned(0, 1, 2)
    backend.set_prefill_mode(mode)
    try:
        for bits in (4, 8):
            for xdt in ("f16", "bf16"):
                for n, K in ((272, 512), (48, 416), (528, 576), (16, 96), (32, 32), (64, 1184)):
                    for ydt in ("f32", "bf16"):
                        _check_up(backend, bits, 2, n, K, T, 1, xdt, ydt, "padded", seed=T)
                _check_up(backend, bits, 2, 160, 672, T, 2, xdt, "bf16", swiglu=True, seed=T)
                _check_down(backend, bits, 2, 272, 416, T, 2, xdt, "bf16", "padded", seed=T)
    finally:
        backend.set_prefill_mode("fast")


@gpu
def test_rounded_operands_where_y_is_rounded_more(backend):
    """FAST mode: a weight of round_f16(scale * q) is off by 2^-11 / sqrt(3) at most on average, 3e-4 on y, next to at most
    2^-8 / sqrt(3) of y's own rounding (both independent from element to element): 2.28e-3 together."""
    E, n, K, T, k = 4, 256, 1024, 200, 2
    w, wd = _stack(backend, 4, E, n, K, 1)
    ids = _ids(T, k, E, 2)
    for xdt in ("bf16", "f16"):
        x = _rows((T, K), xdt, 3)
        ref = _products(x, k, wd, ids)
        y, exact = (torch.empty((T * k, n), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        backend.matmul_experts(w, E, x, ids, y)
        try:
            backend.set_prefill_mode("exact")
            backend.matmul_experts(w, E, x, ids, exact)
        finally:
            backend.set_prefill_mode("fast")
        torch.cuda.synchronize()
        for got, most in ((y, 2.28e-3), (exact, 2.0 ** -8 / 3 ** 0.5)):
            err = ((got.double() - ref).norm() / ref.norm()).item()
            assert err < most, (xdt, err)
        assert not torch.equal(y, exact)
    w.free()


@gpu
def test_rounded_operands_of_rows_of_any_size_and_wide_scales(backend):
    """bf16 rows of 1e-30 and 1e30 become f16 behind a power of two; a weight whose scale * q leaves f16 keeps exact operands."""
    E, n, K, T = 3, 32, 256, 150
    for scale in (0.01, 3.0e4):
        w, wd = _stack(backend, 4, E, n, K, 6, scale)
        size = torch.tensor([1e-30, 1e30 if scale < 1 else 1e25, 1.0, 1e-38], device="cuda").repeat(T)[:T, None]
        x = (_rows((T, K), "f32", 8) * size).bfloat16()
        x[5] = 0
        ids = _ids(T, 1, E, 9)
        y = torch.empty((T, n), dtype=torch.bfloat16, device="cuda")
        backend.matmul_experts(w, E, x, ids, y)
        torch.cuda.synchronize()
        ref = _products(x, 1, wd, ids)
        keep = ref.abs().amax(dim=1) > 1e-36                          # (below, y itself has no bits left)
        assert (y[5] == 0).all()
        _close(y[keep], ref[keep], HALF_STEP["bf16"] + 3e-4, scale)
        w.free()


@gpu
def test_lists_of_many_experts_and_pairs(backend, tuned):
    """1024 experts, 40000 pairs, a third of them with none: against the same products expert by expert."""
    _check_up(backend, 4, 1024, 16, 32, 5000, 8, "f16", "f32", "padded", seed=3)
    tuned(0, 1, 2)
    _check_up(backend, 8, 1024, 16, 64, 5000, 8, "bf16", "f32", "padded", seed=4)
    _check_up(backend, 4, 1, 16, 64, 66000, 1, "f16", "f16", "one", seed=5)


@gpu
@pytest.mark.parametrize("T", [3, 60, 600])
def test_the_same_bits_every_time(backend, T):
    run, _, bufs, _, _ = _layer(backend, T, 16, 4, 256, 160, "bf16", 90)
    run(backend)
    torch.cuda.synchronize()
    first = {n: b.clone() for n, b in bufs.items()}
    for _ in range(3):
        run(backend)
        torch.cuda.synchronize()
        assert all(torch.equal(first[n], b) for n, b in bufs.items())


@gpu
def test_two_contexts_on_two_streams(backend):
    """Each context has scratch of its own: calls of two of them may overlap."""
    other = Backend(0)
    try:
        sides = [torch.cuda.Stream(), torch.cuda.Stream()]
        runs = [_layer(be, 400, 8, 4, 512, 256, "bf16", 100 + i) for i, be in enumerate((backend, other))]
        torch.cuda.synchronize()
        for _ in range(5):
            for (run, *_), be, s in zip(runs, (backend, other), sides):
                run(be, s.cuda_stream)
        torch.cuda.synchronize()
        for _, want, bufs, _, _ in runs:
            _close(bufs["y"], want()[1], 4 * TIGHT + 2 * HALF_STEP["bf16"])
    finally:
        other.close()


def _layer(backend, T, E, k, hidden, width, dt, seed=0):
    gate, gd = _stack(backend, 4, E, width, hidden, seed)
    up, ud = _stack(backend, 4, E, width, hidden, seed + 1)
    pair = backend.fuse_pairs(gate, up)
    down, dd = _stack(backend, 4, E, hidden, width, seed + 2)
    x = _rows((T, hidden), dt, seed + 3)
    logits = _rows((T, E), "f32", seed + 4)
    bufs = {"ids": torch.empty((T, k), dtype=torch.int32, device="cuda"), "w": torch.empty((T, k), device="cuda"),
            "h": torch.empty((T * k, width), dtype=TDT[dt], device="cuda"), "y": torch.empty((T, hidden), dtype=TDT[dt], device="cuda")}

    def run(be, stream=0):
        be.route(logits, bufs["ids"], bufs["w"], score="sigmoid", stream=stream)
        be.matmul_experts(pair, E, x, bufs["ids"], bufs["h"], "swiglu", stream=stream)
        be.matmul_experts_sum(down, E, bufs["h"], bufs["ids"], bufs["w"], bufs["y"], x, stream=stream)

    def want():
        rid, rw = _route_ref(logits.double().cpu().numpy(), k, score="sigmoid")
        ids = torch.from_numpy(rid).cuda()
        g = _products(x, k, gd, ids)
        h = g * torch.sigmoid(g) * _products(x, k, ud, ids)
        z = _products(h, 1, dd, ids) * torch.from_numpy(rw).cuda().reshape(-1, 1)
        return ids, x.double() + z.reshape(T, k, hidden).sum(dim=1)

    return run, want, bufs, x, logits


@gpu
@pytest.mark.parametrize("T", [1, 12, 300])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_a_layer(backend, T, dt):
    """Router, gate and up, down in a row, against the whole in float64.  The rows between the products are rounded once
    to the activations' type, y once more."""
    run, want, bufs, _, _ = _layer(backend, T, 16, 4, 256, 160, dt)
    run(backend)
    torch.cuda.synchronize()
    ids, ref = want()
    assert torch.equal(bufs["ids"], ids)
    _close(bufs["y"], ref, 4 * TIGHT + 2 * HALF_STEP[dt], T)


@gpu
@pytest.mark.parametrize("T,dt", [(1, "f16"), (12, "f16"), (300, "f16"), (300, "bf16")])
def test_a_captured_layer_follows_its_inputs(T, dt):
    """One recording, replayed with other rows and other logits, eager calls of the context between the replays."""
    be = Backend(0)
    try:
        run, want, bufs, x, logits = _layer(be, T, 16, 4, 256, 160, dt, 30)
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):                    # the first launches of this context
            run(be, torch.cuda.current_stream().cuda_stream)
        for i in range(4):
            x.copy_(_rows(tuple(x.shape), dt, 50 + i))
            logits.copy_(_rows(tuple(logits.shape), "f32", 60 + i))
            for b in bufs.values():
                b.fill_(-3)
            graph.replay()
            torch.cuda.synchronize()
            got = {n: b.clone() for n, b in bufs.items()}
            ids, ref = want()
            assert torch.equal(got["ids"], ids)
            _close(got["y"], ref, 4 * TIGHT + 2 * HALF_STEP[dt], i)
            run(be)
            torch.cuda.synchronize()
            assert all(torch.equal(got[n], b) for n, b in bufs.items())      # the same bits as eager calls
    finally:
        be.close()


@gpu
def test_another_stream(backend):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for T in (3, 150):
            run, want, bufs, _, _ = _layer(backend, T, 8, 2, 128, 64, "bf16", 70)
            side.synchronize()
            run(backend, side.cuda_stream)
            side.synchronize()
            _close(bufs["y"], want()[1], 4 * TIGHT + 2 * HALF_STEP["bf16"], T)


# ---- the stack and the driver ----------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("M,dt", [(1, "f16"), (5, "f16"), (260, "bf16")])
def test_a_step_of_the_expert_stack(backend, M, dt):
    """The last layer's calls recomputed in float64 from its dequantised weights and the rows it was given."""
    from cyb_amd import stack
    E, k, hidden, width = 12, 3, 256, 96
    st = stack.build_experts(backend, layers=2, experts=E, top_k=k, hidden=hidden, width=width, seed=3)
    assert len(st.weights) == 10 and len(st.nodes) == 12
    step = stack.stepper(st, M, xdtype=TDT[dt])
    step()
    torch.cuda.synchronize()
    b = step.edges

    def values(w):
        out = torch.empty((w.N, w.K), device="cuda")
        backend.dequant(w, out)
        torch.cuda.synchronize()
        return out.double()

    logits = b["mid"].double() @ values(st.router[-1]).T.contiguous()
    assert ((b["logits"].double() - logits).norm() / logits.norm()).item() < 5e-4
    rid, rw = _route_ref(b["logits"].double().cpu().numpy(), k)
    assert np.array_equal(b["ids"].cpu().numpy(), rid)
    strips = values(st.gate_up[-1]).reshape(E, width // 16, 2, 16, hidden)
    g = _products(b["mid"], k, strips[:, :, 0].reshape(E, width, hidden), b["ids"])
    u = _products(b["mid"], k, strips[:, :, 1].reshape(E, width, hidden), b["ids"])
    _close(b["h"], g * torch.sigmoid(g) * u, 3 * TIGHT + HALF_STEP[dt])
    z = _products(b["h"], 1, values(st.down[-1]).reshape(E, hidden, width), b["ids"]) * torch.from_numpy(rw).cuda().reshape(-1, 1)
    _close(b["y"], b["mid"].double() + z.reshape(M, k, hidden).sum(dim=1), 4 * TIGHT + HALF_STEP[dt])
    with pytest.raises(CybqError):
        stack.build_experts(backend, layers=1, experts=2, top_k=3, hidden=256, width=96)
    for w in st.weights:
        w.free()


@gpu
def test_the_driver_walks_experts(backend):
    from cyb_amd import driver, stack
    st = stack.build_experts(backend, layers=2, experts=8, top_k=2, hidden=256, width=64)
    evs = list(driver.ask(backend, st, prompt_tokens=150, new_tokens=4, chunk=64))
    assert [e["Prefill"]["done"] for e in evs if "Prefill" in e] == [0, 64, 128, 150]
    assert sum("Delta" in e for e in evs) == 4 and evs[-1]["Answer"].tokens == 4
    assert evs[-1]["Answer"].tok_in_s > 0 and evs[-1]["Answer"].tok_out_s > 0
    for w in st.weights:
        w.free()


# ---- refusals ----------------------------------------------------------------------------------------------------

def _status(call):
    with pytest.raises(CybqError) as e:
        call()
    return e.value.status


@gpu
def test_refusals(backend):
    be, lib = backend, backend._lib
    w, _ = _stack(be, 4, 4, 48, 64, 0)
    x = torch.zeros((2, 64), dtype=torch.float16, device="cuda")
    ids = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    g = torch.zeros((2, 2), device="cuda")
    y = torch.zeros((4, 48), device="cuda")
    z = torch.zeros((2, 8), device="cuda")
    assert _status(lambda: be.matmul_experts(w, 4, x, ids.t(), y)) == -2               # not contiguous
    assert _status(lambda: be.matmul_experts(w, 4, x[:1], ids, y)) == -2 and _status(lambda: be.matmul_experts(w, 4, x, ids, y[:3])) == -2
    assert _status(lambda: be.matmul_experts_sum(w, 4, torch.zeros((4, 64), device="cuda"), ids, g, y[:2], y[:2].half())) == -1
    assert _status(lambda: be.route(z, ids, g, bias=torch.zeros(8, device="cuda", dtype=torch.float16))) == -1
    assert _status(lambda: be.set_experts_tuning(3)) == -1
    assert _status(lambda: be.matmul_experts(w, 5, x, ids, y)) == -2                   # 192 rows
    assert _status(lambda: be.matmul_experts(w, 8, x, ids, y)) == -2                   # 24 rows each are no multiple of 16
    assert _status(lambda: be.matmul_experts(w, 0, x, ids, y)) == -2
    assert _status(lambda: be.matmul_experts(w, 1025, x, ids, y)) == -2
    assert _status(lambda: be.matmul_experts(w, 4, x, ids, y, "swiglu")) == -1         # not a pair
    assert _status(lambda: be.matmul_experts(w, 4, x, ids, y, "add")) == -1
    pair = be.fuse_pairs(w, w)
    assert _status(lambda: be.matmul_experts(pair, 8, x, ids, y, "swiglu")) == -2      # gate and up of 24 rows each
    many = torch.zeros((2, 65), dtype=torch.int32, device="cuda")
    assert _status(lambda: be.matmul_experts(w, 4, x, many, torch.zeros((130, 48), device="cuda"))) == -2
    assert _status(lambda: be.route(torch.zeros((3, 8), device="cuda"), ids, g)) == -2
    assert _status(lambda: be.route(z, ids, g, groups=3)) == -2
    assert _status(lambda: be.route(z, ids, g, groups=2, top_groups=3)) == -2
    assert _status(lambda: be.route(z, ids, g, groups=8, top_groups=1)) == -2          # fewer experts than top_k
    assert _status(lambda: be.route(z, ids, g, group_best=3)) == -1
    assert _status(lambda: be.route(torch.zeros((2, 1), device="cuda"), ids, g)) == -2
    assert _status(lambda: be.route(torch.zeros((2, 1025), device="cuda"), ids, g)) == -2
    ctx, wh = be._ctx, w.handle
    p = x.data_ptr()
    assert lib.cybq_matmul_experts(ctx, wh, 4, None, 1, 2, 2, ids.data_ptr(), y.data_ptr(), 0, 0, None) == -1
    assert lib.cybq_matmul_experts(ctx, wh, 4, p, 1, -1, 2, ids.data_ptr(), y.data_ptr(), 0, 0, None) == -2
    assert lib.cybq_matmul_experts(ctx, wh, 4, p, 1, (1 << 24) + 1, 2, ids.data_ptr(), y.data_ptr(), 0, 0, None) == -2
    assert lib.cybq_matmul_experts(ctx, wh, 4, p + 2, 1, 1, 2, ids.data_ptr(), y.data_ptr(), 0, 0, None) == -3
    assert lib.cybq_matmul_experts(ctx, wh, 4, p, 1, 1, 2, ids.data_ptr() + 2, y.data_ptr(), 0, 0, None) == -3
    assert lib.cybq_matmul_experts(ctx, wh, 4, p, 7, 1, 2, ids.data_ptr(), y.data_ptr(), 0, 0, None) == -1
    assert lib.cybq_matmul_experts_sum(ctx, wh, 4, p, 1, 1, 2, ids.data_ptr(), None, None, y.data_ptr(), 0, None) == -1
    assert lib.cybq_route(ctx, z.data_ptr(), 0, 2, 8, 2, 2, None, 1, 1, 1, 1, 1.0, ids.data_ptr(), g.data_ptr(), None) == -1
    for h in (w, pair):
        h.free()


def _blank():
    """A backend and a weight of 4 experts [32, 64] without a device: the checks that come before the library."""
    be = Backend.__new__(Backend)
    be.device, be._addr, be._ctx, be.weights, be._lib = 0, 0, ctypes.c_void_p(), {}, load_library()
    w = QWeight.__new__(QWeight)
    w._h, w._addr, w._backend, w.N, w.K, w.quant = ctypes.c_void_p(), 0, be, 128, 64, formats.Q4
    return be, w


def test_checks_before_the_library():
    be, w = _blank()
    ids, g = torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 2))
    x, y = torch.zeros((2, 64)), torch.zeros((4, 32))
    assert _status(lambda: be.matmul_experts(w, 4, x, ids, y)) == -1                   # not on the device
    assert _status(lambda: be.matmul_experts(w, 4, x, ids.long(), y)) == -2
    assert _status(lambda: be.matmul_experts(w, 4, x, ids.reshape(-1), y)) == -2
    assert _status(lambda: be.matmul_experts(w, 4, x, ids, y, "gelu")) == -1
    assert _status(lambda: be.matmul_experts_sum(w, 4, x, ids, g.double(), y)) == -2
    assert _status(lambda: be.matmul_experts_sum(w, 4, x, ids, g[:1], y)) == -2
    assert _status(lambda: be.route(torch.zeros((2, 8)), ids, g, score="top")) == -1


def test_native_calls_hand_back_what_they_cannot_look_over():
    """Tensors of another device, type or shape are the Python checks' business (1), which answer with an error."""
    from cyb_amd import backend as B
    calls = B._load_calls()
    assert calls
    blank = ctypes.create_string_buffer(4096)
    a = ctypes.addressof(blank)
    x, ids, g, y = torch.zeros((2, 64)), torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 2)), torch.zeros((4, 32))
    for t in (ids, ids.long(), None, 3, ids.reshape(-1)):
        assert calls.experts(a, 0, a, 4, x, t, y, 0, 0) == 1
        assert calls.experts_sum(a, 0, a, 4, x, t, g, y, None, 0) == 1
        assert calls.route(a, 0, x, t, g, 0, None, 1, None, 1, True, 1.0, 0) == 1
    assert calls.experts(0, 0, a, 4, x, ids, y, 0, 0) == 1 and calls.experts(a, 0, a, 0, x, ids, y, 0, 0) == 1 and calls.experts() == 1


def test_no_context():
    lib = load_library()
    assert lib.cybq_route(None, None, 0, 1, 8, 2, 0, None, 1, 1, 1, 1, 1.0, None, None, None) == -1
    assert lib.cybq_matmul_experts(None, None, 4, None, 1, 1, 2, None, None, 0, 0, None) == -1
    assert lib.cybq_matmul_experts_sum(None, None, 4, None, 1, 1, 2, None, None, None, None, 0, None) == -1
