"""The products of a mixture of experts, in every kernel, against the bounds that include/cybq.h states.

Where they come from, u = 2^-24, G = K / 32 groups.  A wave adds at most G scaled group sums one after another: addition g is off by at most
u of a partial sum that has grown like sqrt(g / G) of the whole, evenly spread, so u sqrt(G / 6) of it together (eight waves' sums are joined with a
few u more).  A group's sum is 32 products of integers and 16-bit rows.  The pipe cuts them at u of their largest, next to a sum that is about a fifth
of it (Q4: operands 16 .. 31, bias 24; Q8 0 .. 255, bias 128): 5 u of the group's size and, where the cuts of different groups are independent, of y.
fp32 rows are three such products, whose parts fill all 24 bits, so the results of six MFMAs are cut instead of one or two, always downwards:
this part grows with sqrt(G) as well, and gets the same u sqrt(G) and the doubled constant.  16-bit rows: (4 + sqrt(G)) u, more than twice the chain;
fp32 rows: (8 + 2 sqrt(G)) u.  The operands with a bias of 136 that the first kernels had (2.8e-6 at K = 2048) stay outside both."""
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = 2.0 ** -24


def bound(K, dt):
    root = (K / 32) ** 0.5
    return U * (8 + 2 * root) if dt == "f32" else U * (4 + root)


def stack(be, bits, N, K, seed):
    """N rows of N(0, 0.02) as their quantisation sees them, and the same in float64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    top = 8 if bits == 4 else 128
    q = torch.empty((N, K), device="cuda").normal_(0.0, 3.2 if bits == 4 else 56.0, generator=g).round_().clamp_(-top, top - 1)
    s = ((torch.rand((N, K // 32), device="cuda", generator=g) + 0.5) * (0.0063 if bits == 4 else 0.00036)).half()
    i = q.to(torch.int8)
    i = i[:, 0::2] & 15 | i[:, 1::2] << 4 if bits == 4 else i
    w = be.weight_from_device(bits, N, K, i.contiguous().view(torch.uint8), s.view(torch.int16))
    torch.cuda.synchronize()
    return w, q.double() * s.double().repeat_interleave(32, dim=1)


@pytest.fixture
def tuned(backend):
    yield backend.set_experts_tuning
    backend.set_experts_tuning()


@gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("K", [2048, 14336, 131072])
def test_errors_stay_below_what_the_interface_states(backend, tuned, bits, dt, K):
    n = 64
    w, wd = stack(backend, bits, n, K, K + bits)
    g = torch.Generator(device="cuda").manual_seed(K)
    # one row, a few rows with 1, 4 and 8 waves side by side, tiles of many, token by token
    for path, T, tuning in (("row", 1, (4, 1 << 20, 2)), ("few 1", 12, (1, 1 << 20, 2)), ("few 4", 12, (4, 1 << 20, 2)), ("few 8", 20, (8, 1 << 20, 2)),
                            ("many", 70, (0, 1, 2)), ("token", 5, (0, 0, 1))):
        tuned(*tuning)
        x = torch.empty((T, K), device="cuda").normal_(generator=g).to(TDT[dt])
        ids = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
        y = torch.empty((T, n), device="cuda")
        if path == "token":
            backend.matmul_experts_sum(w, 1, x, ids, torch.ones((T, 1), device="cuda"), y)
        else:
            backend.matmul_experts(w, 1, x, ids, y)
        torch.cuda.synchronize()
        ref = x.double() @ wd.T.contiguous()
        err = ((y.double() - ref).norm() / ref.norm()).item()
        assert err < bound(K, dt), (path, err)
    w.free()


@gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rounded_operands_are_all_that_fast_mode_rounds(backend, bits, dt):
    """Many rows, 16-bit rows, a y of bf16: y is the product of the rows with round_f16(scale * q), rounded once.  Half a step of bf16 for every
    element, and the fp32 sums' share of its row's size (an element may be off by more than the root of the mean square: eight times)."""
    E, n, K, T, k = 4, 256, 1024, 200, 2
    w, wd = stack(backend, bits, E * n, K, bits)
    rounded = wd.to(torch.float16).double().reshape(E, n, K)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty((T, K), device="cuda").normal_(generator=g).to(TDT[dt])
    ids = torch.randint(0, E, (T, k), device="cuda", generator=g).int()
    y = torch.empty((T * k, n), dtype=torch.bfloat16, device="cuda")
    backend.matmul_experts(w, E, x, ids, y)
    torch.cuda.synchronize()
    ref = torch.empty((T * k, n), dtype=torch.float64, device="cuda")
    for e in range(E):
        p = (ids.reshape(-1) == e).nonzero().reshape(-1)
        ref[p] = x.double()[p // k] @ rounded[e].T.contiguous()
    size = ref.square().mean(dim=1, keepdim=True).sqrt()
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 8 * bound(K, dt) * size).all()
    w.free()
