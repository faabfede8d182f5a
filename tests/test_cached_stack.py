"""Cache and attention as they are used: whole layers next to the quantised linears, the driver's conversations, the C++ host layer."""
import os
import subprocess

import numpy as np
import pytest
import torch

from tests.cache_lib import HALF_STEP, TDT, held, turned
from cyb_amd import CybqError

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CACHE_TEST = os.path.join(ROOT, "tests", "cpp", "_build", "cache_test")
NAMES = {v: k for k, v in TDT.items()}


class Recorder:
    """A backend that keeps copies of what its calls were given and gave."""

    def __init__(self, be):
        self._be, self.calls = be, []

    def __getattr__(self, name):
        f = getattr(self._be, name)
        if name not in ("matmul_norm", "matmul_ex", "cache_append", "attention"):
            return f

        def call(*a, **kw):
            copy = lambda t: t.clone() if isinstance(t, torch.Tensor) else t
            before = [copy(t) for t in a]
            f(*a, **kw)
            torch.cuda.synchronize()
            self.calls.append((name, before, [copy(t) for t in a]))
        return call


def _close(got, want, size, rounding):
    """|got - want| <= its own rounding of |want| and what sums of terms of `size` lose on the way (2^-16 of it)."""
    err, bound = (got.double() - want).abs(), (rounding + 2.0 ** -20) * want.abs() + size + 2.0 ** -24
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.2f} bounds"


def _values(be, w):
    out = torch.empty((w.N, w.K), device="cuda")
    be.dequant(w, out)
    torch.cuda.synchronize()
    return out.double()


def _linear(x, w):
    """x W^T in float64, and the sums of |x| |w|."""
    return x @ w.T.contiguous(), x.abs() @ w.abs().T.contiguous()


@gpu
@pytest.mark.parametrize("kind,dt,window", [("q8", "f16", 0), ("q4", "bf16", 40), ("f16", "bf16", 0), ("bf16", "bf16", 33)])
def test_whole_layers(backend, kind, dt, window):
    """Two conversations read a prompt in two chunks and go on together for three tokens; every call of the layers is recomputed in float64 from
    what it was given, the cache's contents included.

    Rows of more than 32 go through kernels that round a weight, and the row, once to f16: each product is off by 2^-11 + 2^-11 and a little,
    2^-10 (1 + 2^-6) of sum |x| |w|; few rows are exact up to fp32 sums (2^-16 leaves room for K = 512 of them).  A folded norm scales x by gamma in
    fp32 and rounds it to the operand's type (bf16 rows of the few: 2^-8).  Attention: y's rounding, p's and (many rows) the values' to the
    operand's type, keys' the same way through their scores: 2 eps sum |q| |k| scale on an exponent."""
    from cyb_amd import stack
    heads, kvh, dim, rounding = 8, 2, 64, HALF_STEP[dt]
    st = stack.build_cached(backend, layers=2, kind=kind, conversations=2, context=130, heads=heads, kv_heads=kvh, head_dim=dim, width=320, page=32,
                            window=window, seed=11)
    assert len(st.nodes) == 12 and len(st.weights) == 8 and st.conversations == 2
    st.backend = rec = Recorder(backend)
    group = heads // kvh
    layers, held_k, held_v = 2, {}, {}
    plan = [(1, 41, 0), (1, 41, 1), (1, 7, 0), (1, 7, 1), (2, 2, 0), (2, 2, 0), (2, 2, 0)]
    position = [0, 0]
    for count, M, first in plan:
        step = st.stepper(M, TDT[dt], count=count, seed=M + first)
        rec.calls.clear()
        step(0, first)
        torch.cuda.synchronize()
        n, where = M // count, []
        for c in range(first, first + count):
            where += [(c, position[c] + i) for i in range(n)]
            position[c] += n
        assert st.lengths.tolist() == position
        assert [c[0] for c in rec.calls] == ["matmul_norm", "cache_append", "attention", "matmul_ex", "matmul_norm", "matmul_ex"] * layers
        loose = (2.0 ** -10 * (1 + 2.0 ** -6) if M > 2 else 2.0 ** -16)
        x = step.edges["x"]
        for i in range(layers):
            (_, a, got), (_, append, appended), (_, att, attended), (_, oa, og), (_, ga, gg), (_, da, dg) = rec.calls[6 * i:6 * i + 6]
            assert torch.equal(a[1], x)
            # norm + qkv
            def normed(rows, gamma):
                rows = rows.double()
                return rows * gamma.double() / torch.sqrt((rows * rows).mean(dim=1, keepdim=True) + st.eps)
            folded = loose + (rounding if M <= 32 else 0.0)
            want, size = _linear(normed(a[1], st.norms[i][0]), _values(backend, st.qkv[i]))
            _close(got[4], want, folded * size, rounding)
            # the cache: q turned, k and v as a cache of this kind holds them
            qkv = got[4].view(M, heads + 2 * kvh, dim)
            q, k, v = qkv.split([heads, kvh, kvh], dim=1)
            at = torch.tensor([p for _, p in where])
            _close(appended[6], turned(q, at, st.rope, "halves").double(), 0.0, HALF_STEP[NAMES[appended[6].dtype]])
            kk, vv = held(kind, turned(k, at, st.rope, "halves")), held(kind, v.float())
            for r, (c, p) in enumerate(where):
                held_k[i, c, p], held_v[i, c, p] = kk[r], vv[r]
            k_read, v_read = (torch.empty((M, kvh, dim), device="cuda") for _ in range(2))
            backend.cache_read(st.cache, i, append[2], k_read, v_read)
            torch.cuda.synchronize()
            assert torch.equal(k_read.double(), kk) and torch.equal(v_read.double(), vv)
            # attention
            eps = HALF_STEP["bf16" if NAMES[att[3].dtype] == "bf16" else "f16"]
            for r, (c, p) in enumerate(where):
                seen = range(max(0, p - window + 1) if window else 0, p + 1)
                K, V = torch.stack([held_k[i, c, j] for j in seen]), torch.stack([held_v[i, c, j] for j in seen])
                for h in range(heads):
                    qq = att[3][r, h].double()
                    s = K[:, h // group] @ qq * dim ** -0.5
                    soft = torch.softmax(s, dim=0)
                    size = soft @ V[:, h // group].abs()
                    shift = ((K[:, h // group].abs() @ qq.abs()) * dim ** -0.5).max().item()
                    _close(attended[4][r, h], soft @ V[:, h // group], (2 * eps + 2 * (2 * eps * shift) + 2.0 ** -16) * size, eps)
            # o + residual, norm + gate / up + swiglu, down + residual
            want, size = _linear(oa[1].double(), _values(backend, st.o[i]))
            _close(og[2], want + a[1].double(), loose * size, rounding)
            strips = _values(backend, st.gate_up[i]).reshape(-1, 2, 16, st.hidden)
            (g, gs), (u, us) = (_linear(normed(ga[1], st.norms[i][1]), strips[:, e].reshape(-1, st.hidden)) for e in range(2))
            _close(gg[4], g * torch.sigmoid(g) * u, folded * (1.2 * gs * (u.abs() + folded * us) + us * g.abs()) + 2.0 ** -18 * (g * u).abs(), rounding)
            want, size = _linear(da[1].double(), _values(backend, st.down[i]))
            _close(dg[2], want + da[4].double(), loose * size, rounding)
            x = dg[2]
        assert torch.equal(step.edges["y"], x)
    # the same again from the start: the same bits
    last = x.clone()
    st.backend = backend
    st.set_lengths(0)
    for count, M, first in plan:
        step = st.stepper(M, TDT[dt], count=count, seed=M + first)
        step(0, first)
    torch.cuda.synchronize()
    assert torch.equal(step.edges["y"], last)
    with pytest.raises(CybqError):
        st.stepper(3, count=2)
    with pytest.raises(CybqError):
        st.stepper(2, count=2)(0, 1)
    st.free()


@gpu
def test_a_captured_step_goes_on(backend):
    """One token's step through two layers in a graph: each replay is the next token, as eager steps are."""
    from cyb_amd import stack
    st = stack.build_cached(backend, layers=2, kind="q8", conversations=3, context=70, heads=4, kv_heads=2, head_dim=64, width=256, page=32, seed=12)
    prompt = st.stepper(40)
    one = st.stepper(3, count=3)
    outs = []
    for c in range(3):
        prompt(0, c)
    for _ in range(6):
        one()
        torch.cuda.synchronize()
        outs.append(one.edges["y"].clone())
    st.set_lengths(0)
    for c in range(3):
        prompt(0, c)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one(torch.cuda.current_stream().cuda_stream)
    for i in range(6):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(one.edges["y"], outs[i]), i
        assert st.lengths.tolist() == [41 + i] * 3
    st.free()


@gpu
def test_the_driver_keeps_a_cache(backend):
    from cyb_amd import driver, stack
    st = stack.build_cached(backend, layers=2, kind="q4", conversations=2, context=80, heads=4, kv_heads=2, head_dim=64, width=256)
    evs = list(driver.ask(backend, st, prompt_tokens=50, new_tokens=4, chunk=32, batch=2))
    assert [e["Prefill"]["done"] for e in evs if "Prefill" in e] == [0, 32, 50, 82, 100]
    assert evs[-1]["Answer"].tokens == 8 and evs[-1]["Answer"].tok_in_s > 0 and evs[-1]["Answer"].tok_out_s > 0
    assert st.lengths.tolist() == [54, 54]
    assert len(list(driver.ask(backend, st, prompt_tokens=0, new_tokens=3, batch=1))) == 5 and st.lengths.tolist() == [3, 0]
    with pytest.raises(ValueError):
        list(driver.ask(backend, st, prompt_tokens=76, new_tokens=4))
    with pytest.raises(ValueError):
        list(driver.ask(backend, st, prompt_tokens=5, new_tokens=4, batch=3))
    st.free()


def test_cpp_without_a_device():
    if not os.path.exists(CACHE_TEST):
        pytest.fail("tests/cpp/_build/cache_test missing: run __graft_entry__.build()")
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    out = subprocess.run([CACHE_TEST, "--refusals"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout == "made 0 held 0 read -1 attention -1\n", out.stdout + out.stderr


@gpu
def test_cpp_cache():
    if not os.path.exists(CACHE_TEST):
        pytest.fail("tests/cpp/_build/cache_test missing: run __graft_entry__.build()")
    out = subprocess.run([CACHE_TEST, "--run"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("stored same"), out.stdout + out.stderr


@gpu
def test_the_driver_on_a_stream_of_its_own(backend):
    """Lengths that are set late - work is in front of them on the stream that they are set on - are there for the steps that count on them."""
    from cyb_amd import driver, stack
    st = stack.build_cached(backend, layers=1, kind="q8", conversations=2, context=80, heads=4, kv_heads=2, head_dim=64, width=256)
    starts, lengths = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 53, 106], [53, 53]))
    batch, kept = backend.cache_batch(starts, lengths, st.tables, 106), []
    side, set_now = torch.cuda.Stream(), st.set_lengths

    def set_late(*args):
        torch.cuda._sleep(20_000_000)
        set_now(*args)
    st.set_lengths = set_late
    for stream in (0, side.cuda_stream):
        evs = list(driver.ask(backend, st, prompt_tokens=50, new_tokens=3, chunk=32, batch=2, stream=stream))
        torch.cuda.synchronize()
        assert st.lengths.tolist() == [53, 53] and evs[-1]["Answer"].tokens == 6
        kv = [torch.empty((106, 2, 64), device="cuda") for _ in range(2)]
        backend.cache_read(st.cache, 0, batch, *kv)
        torch.cuda.synchronize()
        kept.append(kv)
        st.set_lengths(80)
    assert torch.equal(kept[0][0], kept[1][0]) and torch.equal(kept[0][1], kept[1][1])
    st.free()


@gpu
def test_lengths_are_counted_on_the_stacks_device(backend, monkeypatch):
    """A step's own torch work goes to its stream on the backend's device, whichever device is the current one."""
    from cyb_amd import stack
    st = stack.build_cached(backend, layers=1, kind="q8", conversations=1, context=40, heads=2, kv_heads=1, head_dim=64, width=64, page=32)
    step, side, made = st.stepper(1), torch.cuda.Stream(), []
    torch.cuda.synchronize()
    stream_of = torch.cuda.ExternalStream
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda *a, **kw: made.append((a, kw)) or stream_of(*a, **kw))
    step(side.cuda_stream)
    torch.cuda.synchronize()
    assert made == [((side.cuda_stream,), {"device": backend.device})] and st.lengths.tolist() == [1]
    st.free()
