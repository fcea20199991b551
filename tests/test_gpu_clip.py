"""Global gradient norm and clipping against the definition in 64 bits and torch's function of the same name."""

import math

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import _capi as C
from prime_rl_cse_amd import optim

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F = torch.bfloat16, torch.float32


def params(shapes, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for shape, dtype in shapes:
        p = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
        p.grad = (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)
        out.append(p)
    return out


def check(ps, max_norm, norm_type=2.0):
    before = [p.grad.clone() for p in ps if p.grad is not None]
    flat = torch.cat([g.double().reshape(-1) for g in before])
    want = flat.norm() if norm_type == 2.0 else flat.abs().max()
    got = optim.clip_grad_norm_(ps, max_norm, norm_type)
    assert got.dtype == F and got.shape == ()
    # squares added in fp64, the root rounded once to fp32
    assert abs(float(got) - float(want)) <= 2.0**-24 * (1 + 1e-6) * float(want)
    coef = min(1.0, max_norm / (float(want) + 1e-6))
    for p, g in zip((p for p in ps if p.grad is not None), before):
        if max_norm >= float(want) * (1 + 2.0**-20) + 2e-6:
            assert torch.equal(p.grad, g)
            continue
        # the factor: norm, its sum with 1e-6 and the quotient rounded, the product once more, then to the type
        ref = g.double() * coef
        tol = ref.abs() * (4 * 2.0**-24 + (2.0**-8 if g.dtype == BF else 0.0)) + 2.0**-149
        assert bool(((p.grad.double() - ref).abs() <= tol).all())
    return got


SHAPES = {
    "one element": [((1,), F)],
    "one bf16 element": [((), BF)],
    "small": [((3, 5), F), ((7,), BF), ((1, 1, 9), F), ((0, 4), F), ((8,), BF)],
    "a chunk and one": [((8192,), F), ((8193,), BF), ((8191,), F)],
    "many": [((1 + 37 * i % 911,), BF if i % 3 else F) for i in range(411)],
    "larger": [((1021, 2053), F), ((4099, 1013), BF), ((1 << 22,), BF)],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.25, 1e9])
@pytest.mark.parametrize("which", list(SHAPES))
def test_against_the_definition(which, max_norm, norm_type):
    a, b = params(SHAPES[which]), params(SHAPES[which])
    n1, n2 = check(a, max_norm, norm_type), optim.clip_grad_norm_(b, max_norm, norm_type)
    assert torch.equal(n1, n2) and all(torch.equal(p.grad, q.grad) for p, q in zip(a, b))  # same inputs, same bits


def test_agrees_with_torch():
    a, b = params([((300, 70), F), ((11,), F)]), params([((300, 70), F), ((11,), F)])
    n1, n2 = optim.clip_grad_norm_(a, 1.0), torch.nn.utils.clip_grad_norm_(b, 1.0)
    assert torch.allclose(n1, n2, rtol=1e-6)
    for p, q in zip(a, b):
        assert torch.allclose(p.grad, q.grad, rtol=1e-6, atol=0)
    assert torch.equal(optim.grad_norm([p.grad for p in a]), optim.clip_grad_norm_(a, 1e30))


@pytest.mark.parametrize("dtype", [BF, F])
def test_pieces_of_one_buffer_at_odd_places(dtype):
    gen = torch.Generator(device=DEV).manual_seed(5)
    flat = torch.randn(70001, generator=gen, device=DEV).to(dtype)
    cuts = [(1, 4), (5, 5), (5, 12), (13, 30), (31, 8300), (8300, 16500), (20001, 69999)]  # some touch, some do not
    ps = []
    for a, z in cuts:
        p = torch.zeros(z - a, dtype=dtype, device=DEV, requires_grad=True)
        p.grad = flat[a:z]
        ps.append(p)
    was = flat.clone()
    check([ps[i] for i in (3, 0, 6, 1, 2, 5, 4)], 0.5)
    between = torch.ones(70001, dtype=torch.bool, device=DEV)
    for a, z in cuts:
        between[a:z] = False
    assert torch.equal(flat[between], was[between])


def test_transposed_gradient_and_missing_ones():
    ps = params([((64, 40), F), ((9,), F), ((5,), F)])
    ps[0].grad = ps[0].grad.t().contiguous().t()
    ps[1].grad = None
    check(ps, 0.1)
    assert float(optim.clip_grad_norm_([ps[1]], 1.0)) == 0.0 and float(optim.clip_grad_norm_([], 1.0)) == 0.0
    check(params([((0,), F), ((4,), F)])[1:], 0.1)
    assert float(optim.clip_grad_norm_(params([((0,), F)]), 1.0)) == 0.0
    one = params([((6,), F)])[0]
    assert float(optim.clip_grad_norm_(one, 0.5)) > 0


def test_large_and_tiny_values():
    check(params([((5000,), F)], scale=1e30), 1.0)  # squares beyond fp32
    check(params([((5000,), F)], scale=1e-30), 1.0)  # squares below it
    p = params([((5000,), F)], scale=1e-30)
    assert float(optim.grad_norm([q.grad for q in p])) > 0


def test_what_is_not_finite_does_what_torch_does():
    for bad, norm_type in ((math.nan, 2.0), (math.nan, math.inf), (math.inf, 2.0), (-math.inf, math.inf)):
        for at in (0, 12000, 20000):
            a, b = params([((20001,), F), ((33,), BF)]), params([((20001,), F), ((33,), BF)])
            for ps in (a, b):
                ps[0].grad[at] = bad
            n1, n2 = optim.clip_grad_norm_(a, 1.0, norm_type), torch.nn.utils.clip_grad_norm_(b, 1.0, norm_type)
            assert (math.isnan(float(n1)), math.isinf(float(n1))) == (math.isnan(float(n2)), math.isinf(float(n2)))
            for p, q in zip(a, b):
                assert torch.equal(p.grad.isnan(), q.grad.isnan()) and torch.equal(p.grad.nan_to_num(), q.grad.nan_to_num())
    ps = params([((10,), F)])
    ps[0].grad[3] = math.inf
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert bool((ps[0].grad.isinf().sum() == 1).all())  # refused before anything was scaled


def test_refusals():
    ps = params([((6, 4), F), ((4,), F)])
    with pytest.raises(ValueError):
        optim.clip_grad_norm_([ps[0], ps[0]], 1.0)
    p = torch.zeros(5, device=DEV, requires_grad=True)
    p.grad = ps[0].grad.view(-1)[3:8]
    with pytest.raises(ValueError):
        optim.clip_grad_norm_([ps[0], p], 1.0)
    for g in (torch.ones(1, device=DEV).expand(5), torch.ones(10, device=DEV)[::2]):
        p.grad = g
        assert not optim.clip_grad_norm_supported([g])
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], 1.0)
    h = torch.zeros(5, device=DEV, dtype=torch.half, requires_grad=True)
    h.grad = torch.ones_like(h)
    with pytest.raises(ValueError):
        optim.clip_grad_norm_([h], 1.0)
    with pytest.raises(ValueError):
        optim.clip_grad_norm_(ps, 1.0, norm_type=3.0)
    assert optim.clip_grad_norm_supported([q.grad for q in ps])


def test_captured_and_replayed():
    ps = params([((9000,), F), ((1000, 70), BF), ((3,), F)])
    fresh = [p.grad.clone() for p in ps]

    def run():
        for p, g in zip(ps, fresh):
            p.grad.copy_(g)
        return optim.clip_grad_norm_(ps, 2.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run()
    for i in range(3):
        for g in fresh:
            g.normal_(std=0.001 if i == 1 else 1.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [norm.clone(), *(p.grad.clone() for p in ps)]
        want = [run(), *(p.grad for p in ps)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_total_that_ranks_have_added_up():
    g = params([((5000,), F)])[0].grad
    pieces = optim._pieces([g], True)
    table, n = pieces.ctypes.data, len(pieces)
    lib, st = C.load(), C.stream_ptr(g.device)
    ws = torch.empty(lib.prl_grad_norm_workspace_bytes(table, n) // 8, dtype=torch.float64, device=DEV)
    total, out = torch.empty(1, dtype=torch.float64, device=DEV), torch.empty(2, device=DEV)
    C.check(lib.prl_grad_norm(table, n, C.NORM_L2, 1.0, total.data_ptr(), None, None, ws.data_ptr(), ws.numel() * 8, st), "norm")
    both = total * 2  # as if a second rank held the same shard
    C.check(lib.prl_grad_norm_finish(both.data_ptr(), 1, C.NORM_L2, 1.0, None, out.data_ptr(), out.data_ptr() + 4, st), "finish")
    want = g.double().norm() * math.sqrt(2.0)
    assert abs(float(out[0]) - float(want)) <= 2.0**-23 * float(want)
    assert abs(float(out[1]) - 1.0 / (float(want) + 1e-6)) <= 2.0**-22 / float(want)


@pytest.mark.parametrize("which", ["small", "many", "larger"])
def test_one_call_and_its_two_halves_agree(which):
    a, b = params(SHAPES[which]), params(SHAPES[which])
    n1 = optim.clip_grad_norm_(a, 0.5)
    n2 = optim.clip_grad_norm_(b, 0.5, error_if_nonfinite=True)
    assert torch.equal(n1, n2) and all(torch.equal(p.grad, q.grad) for p, q in zip(a, b))


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_one_gradient_of_more_than_2_31_elements(norm_type):
    n = 2**31 + 8195
    p = torch.empty(n, dtype=BF, device=DEV, requires_grad=True)
    p.grad = torch.full((n,), 0.5, dtype=BF, device=DEV)
    p.grad[-1] = -2.0  # the last element alone is the largest
    want = math.sqrt((n - 1) * 0.25 + 4.0) if norm_type == 2.0 else 2.0
    got = optim.clip_grad_norm_(p, want / 2, norm_type)
    assert abs(float(got) - want) <= 2.0**-24 * (1 + 1e-6) * want
    # halves but for 1e-6 and a few fp32 roundings, which bf16's step of 2^-8 hides
    for cut in (slice(0, 9000), slice(2**31 - 9000, 2**31 + 8194)):
        assert bool((p.grad[cut] == 0.25).all())
    assert float(p.grad[-1]) == -1.0
