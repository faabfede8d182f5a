"""Calls of the mixture-of-experts operators that meet the limits of a context's scratch, of a capture and of their arguments."""
import pytest

from cyb_amd.backend import Backend, CybqError

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def planes(bits, N, K, seed):
    """A quantised tensor on the device (q, scales) and its float64 values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (N * K * bits // 8,), dtype=torch.uint8, device="cuda", generator=g)
    s = (0.01 * (0.5 + torch.rand((N, K // 32), device="cuda", generator=g))).half()
    v = torch.stack([q & 15, q >> 4], dim=1).reshape(N, K).double() if bits == 4 else q.view(torch.int8).reshape(N, K).double()
    v = torch.where(v >= 8, v - 16, v) if bits == 4 else v
    return q, s.view(torch.int16), v * s.double().repeat_interleave(32, dim=1)


def normal(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(generator=g).to(dtype)


def products(x, xdiv, wd, ids):
    """float64 [P, n], zeros for pairs without an expert."""
    flat = ids.reshape(-1).long()
    out = torch.zeros((flat.numel(), wd.shape[1]), dtype=torch.float64, device="cuda")
    for e in range(wd.shape[0]):
        p = torch.nonzero(flat == e).reshape(-1)
        if p.numel():
            out[p] = x.double()[p // xdiv] @ wd[e].T.contiguous()
    return out


@gpu
def test_rounds_that_the_scratch_sets(backend):
    """4096 tokens x 8 x 2048 outputs: 268 MB of sums, more than the scratch has; with them the lists, the staged rows and their factors.  The last round
    has fewer pairs than the kernel for many rows takes for 200 experts.  The decode kernels' tickets behind it all are zero at rest, and stay so."""
    E, n, K, T, k = 200, 2048, 160, 4096, 8
    q, s, wd = planes(4, E * n, K, 1)
    w = backend.weight_from_device(4, E * n, K, q, s)
    dq, ds, _ = planes(4, 4096, 4096, 2)
    dense = backend.weight_from_device(4, 4096, 4096, dq, ds)
    one = normal((1, 4096), 3, torch.float16)
    before, after = (torch.empty((1, 4096), device="cuda") for _ in range(2))
    backend.matmul(dense, one, before)
    ids = torch.randint(0, E, (T, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).int()
    ids[T - 300:][torch.rand((300, k), device="cuda") < 0.3] = -1
    ids[T - 7:] = E
    x, residual = normal((T * k, K), 5), normal((T, n), 6)
    g = torch.rand((T, k), device="cuda")
    y = torch.full((T + 1, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    backend.matmul_experts_sum(w, E, x, ids, g, y[:T], residual)
    backend.matmul(dense, one, after)
    torch.cuda.synchronize()
    assert torch.isnan(y[T]).all() and torch.equal(y[T - 7:T], residual[T - 7:]) and torch.equal(before, after)
    z = products(x, 1, wd.reshape(E, n, K), ids) * g.double().reshape(-1, 1)
    z = z.reshape(T, k, n)
    ref = residual.double() + z.sum(dim=1)
    # weights rounded to f16 (2^-11 at most), y to bf16 (2^-8): of the products' and of y's size
    size = z.square().sum(dim=(1, 2)).sqrt() * 2.0 ** -11 + ref.norm(dim=1) * 2.0 ** -8
    assert ((y[:T].double() - ref).norm(dim=1) <= size).all()
    # the same tokens in calls that fit one round: the same bits, where the kernel is the same (the first round's)
    some = torch.empty((1500, n), dtype=torch.bfloat16, device="cuda")
    backend.matmul_experts_sum(w, E, x[:1500 * k], ids[:1500], g[:1500], some, residual[:1500])
    torch.cuda.synchronize()
    assert torch.equal(some, y[:1500])
    for h in (w, dense):
        h.free()


@gpu
@pytest.mark.parametrize("down", [False, True])
def test_the_first_call_on_a_weight_may_sit_in_a_capture(down):
    """Rounded operands hang on the scan of the weight's scales, which a stack made from device memory has not been asked for before its first call."""
    be = Backend(0)
    try:
        E, n, K, T, k = 4, 64, 256, 150, 2
        q, s, wd = planes(4, E * n, K, 7)
        w = be.weight_from_device(4, E * n, K, q, s)
        torch.cuda.synchronize()
        ids = torch.randint(0, E, (T, k), device="cuda").int()
        x, g = normal((T * k if down else T, K), 8), torch.rand((T, k), device="cuda")
        y = torch.zeros((T if down else T * k, n), dtype=torch.bfloat16, device="cuda")

        def call(stream=0):
            if down:
                be.matmul_experts_sum(w, E, x, ids, g, y, stream=stream)
            else:
                be.matmul_experts(w, E, x, ids, y, stream=stream)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            call(torch.cuda.current_stream().cuda_stream)
        for i in range(3):
            x.copy_(normal(tuple(x.shape), 10 + i))
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            call()
            torch.cuda.synchronize()
            assert torch.equal(got, y)
            ref = products(x, 1 if down else k, wd.reshape(E, n, K), ids)
            if down:
                ref = (ref * g.double().reshape(-1, 1)).reshape(T, k, n).sum(dim=1)
            assert ((got.double() - ref).norm() / ref.norm()).item() < 2.0 ** -8 + 2.0 ** -11
        w.free()
    finally:
        be.close()


@pytest.fixture
def tuned(backend):
    yield backend.set_experts_tuning
    backend.set_experts_tuning()


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [32, 768, 1312, 4096])
@pytest.mark.parametrize("bits", [4, 8])
def test_pairs_without_an_expert_take_no_part_token_by_token(backend, tuned, bits, K, dt):
    """A token's absent pairs leave no trace: the same bits as a call of the pairs that are there alone, whatever stands in the others' rows and weights."""
    E, n, k = 9, 48, 8
    q, s, _ = planes(bits, E * n, K, 11)
    w = backend.weight_from_device(bits, E * n, K, q, s)
    tuned(0, 0, 1)
    for there in ([], [0], [7], [1, 4], [0, 2, 5], [1, 3, 4, 6, 7], list(range(8))):
        T, j = 3, torch.tensor(there, dtype=torch.long, device="cuda")
        x = normal((T, k, K), 12, dt)
        ids = torch.randint(0, E, (T, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(13)).int()
        g, residual = torch.rand((T, k), device="cuda"), normal((T, n), 14, torch.float32)
        want = residual.clone()
        if there:
            backend.matmul_experts_sum(w, E, x[:, j].reshape(-1, K).contiguous(), ids[:, j].contiguous(), g[:, j].contiguous(), want, residual)
        absent = torch.tensor([i for i in range(k) if i not in there], dtype=torch.long, device="cuda")
        ids[:, absent], g[:, absent], x[:, absent] = -1, float("nan"), float("inf")
        ids[1, absent] = E
        y = torch.full((T, n), float("nan"), device="cuda")
        backend.matmul_experts_sum(w, E, x.reshape(-1, K), ids, g, y, residual)
        torch.cuda.synchronize()
        assert torch.equal(y, want), there
    w.free()


@gpu
def test_the_router_s_scale_is_finite(backend):
    """Times a score of 0 an infinite scale would be NaN, which weights never are; rows without any score are what it would show in."""
    z = torch.full((3, 8), float("-inf"), device="cuda")
    ids, w = torch.full((3, 2), -5, dtype=torch.int32, device="cuda"), torch.full((3, 2), -5.0, device="cuda")
    for scale in (float("inf"), float("-inf"), float("nan"), 1e300):                  # (1e300 is infinite as a float)
        with pytest.raises(CybqError) as e:
            backend.route(z, ids, w, scale=scale)
        assert e.value.status == -1
        torch.cuda.synchronize()
        assert (ids == -5).all() and (w == -5).all()
    backend.route(z, ids, w, scale=3.4e38)
    torch.cuda.synchronize()
    assert (w == 0).all() and (ids.cpu() == torch.tensor([0, 1])).all()


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_logit_without_a_score_and_a_bias(backend, score):
    """-inf and NaN score 0: behind all others without a bias, c = bias with one; a bias of -inf keeps an expert out."""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[-inf, 0.0, nan, 0.5, 0.25, -3.0]], device="cuda")
    bias = torch.tensor([2.0, 0.0, 3.0, -inf, 0.0, 0.0], device="cuda")
    ids, w = torch.empty((1, 6), dtype=torch.int32, device="cuda"), torch.empty((1, 6), device="cuda")
    backend.route(z, ids, w, score=score)
    torch.cuda.synchronize()
    assert ids.tolist() == [[3, 4, 1, 5, 0, 2]] and w[0, 4:].tolist() == [0.0, 0.0] and (w[0, :4] > 0).all()
    backend.route(z, ids, w, score=score, bias=bias)
    torch.cuda.synchronize()
    assert ids.tolist() == [[2, 0, 4, 1, 5, 3]] and w[0, :2].tolist() == [0.0, 0.0] and (w[0, 2:] > 0).all()
