"""Rotary embedding from position ids against its definition in 64 bits."""

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import _capi as C
from prime_rl_cse_amd import fused

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def turned(x, theta, amplitude, r, interleaved):
    """(the rotated head in float64, |u| + |v| of each element's pair)."""
    x = x.double()
    u, v = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])
    c, s = torch.cos(theta) * amplitude, torch.sin(theta) * amplitude
    a, b, m = u * c - v * s, v * c + u * s, u.abs() + v.abs()
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat([p, q], -1))
    return torch.cat([join(a, b), x[..., r:]], -1), torch.cat([join(m, m), torch.zeros_like(x[..., r:])], -1)


def check(got, x, theta, amplitude, r, interleaved):
    want, m = turned(x, theta, amplitude, r, interleaved)
    # cos and sin: the fraction of a turn rounded to fp32 (at most 2^-25 half turns, pi 2^-25 of angle) and 2 steps of
    # sincospi; the amplitude's product, the two products and the sum: 4 roundings of at most |u| + |v|
    tol = amplitude * m * (3.15 * 2.0**-25 + 2 * 2.0**-23 + 4 * 2.0**-24) + HALF_STEP[x.dtype] * want.abs()
    # this reference rounds the angle itself to 64 bits: 2^-53 of it, 1e-6 rad at position 2^33
    far = theta.abs() * 2.0**-53
    far = far.repeat_interleave(2, -1) if interleaved else torch.cat([far, far], -1)
    tol[..., :r] += amplitude * m[..., :r] * far
    assert got.dtype == x.dtype and got.shape == x.shape
    worst = float(((got.detach().double() - want).abs() / (tol + 1e-300)).max())
    assert worst <= 1.0, worst
    assert torch.equal(got[..., r:], x[..., r:])


def inputs(b, t, hq, hk, d, dtype, layout, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    if layout == "bhtd":
        return mk(b, hq, t, d), mk(b, hk, t, d)
    if layout == "bthd":
        return mk(b, t, hq, d).transpose(1, 2), mk(b, t, hk, d).transpose(1, 2)
    if layout == "stacked":
        y = mk(b, t, hq + 2 * hk, d)
        return y[:, :, :hq].transpose(1, 2), y[:, :, hq : hq + hk].transpose(1, 2)
    if layout == "shifted":  # one element off any alignment, rows of odd pitch
        y = mk(b * (hq + hk) * t * (d + 3) + 1)[1:].view(b, hq + hk, t, d + 3)[..., 1 : d + 1]
        return y[:, :hq], y[:, hq:]
    y = mk(b, hq + hk, t, 2 * d)[..., ::2]  # a stride along the head
    return y[:, :hq], y[:, hq:]


SHAPES = [  # b, t, hq, hk, d, r, layout
    (1, 1, 1, 1, 2, 2, "bhtd"),
    (1, 1, 16, 8, 128, 128, "bthd"),
    (48, 1, 16, 8, 128, 128, "bthd"),
    (2, 37, 4, 2, 64, 32, "bhtd"),
    (1, 300, 14, 2, 64, 64, "stacked"),
    (3, 65, 5, 1, 80, 20, "bthd"),
    (2, 31, 3, 1, 17, 6, "bhtd"),
    (1, 9, 2, 2, 130, 130, "shifted"),
    (2, 5, 2, 1, 96, 34, "shifted"),
    (1, 7, 2, 1, 48, 24, "strided"),
    (1, 3, 1, 1, 700, 516, "bhtd"),
    (1, 2053, 28, 4, 128, 64, "stacked"),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype, interleaved):
    b, t, hq, hk, d, r, layout = shape
    q, k = inputs(b, t, hq, hk, d, dtype, layout)
    q.requires_grad_(True), k.requires_grad_(True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    pos = torch.randint(0, 100000, (b, t), generator=gen, device=DEV)
    inv_freq, amplitude = fused.rope_frequencies(r, 1e6, {"rope_type": "yarn", "factor": 4.0,
                                                          "original_max_position_embeddings": 32768}, device=DEV)
    qo, ko = fused.rope_at_positions(q, k, pos, inv_freq, interleaved=interleaved, attention_scaling=amplitude)
    theta = (pos.double()[..., None] * inv_freq.double())[:, None]
    check(qo, q.detach(), theta, amplitude, r, interleaved)
    check(ko, k.detach(), theta, amplitude, r, interleaved)
    gq, gk = inputs(b, t, hq, hk, d, dtype, layout, seed=2)
    torch.autograd.backward([qo, ko], [gq, gk])
    check(q.grad, gq, -theta, amplitude, r, interleaved)
    check(k.grad, gk, -theta, amplitude, r, interleaved)
    # the gradient against differences of the definition: (f(x + e) - f(x - e)) / 2e along a direction
    dq = torch.randn(q.shape, generator=gen, device=DEV, dtype=torch.float64)
    e = 1e-4
    f = lambda z: (turned(z, theta, amplitude, r, interleaved)[0] * gq.double()).sum()
    slope = (f(q.detach().double() + e * dq) - f(q.detach().double() - e * dq)) / (2 * e)
    got = (q.grad.double() * dq).sum()
    scale = (gq.double().abs() * dq.abs()).sum() * 2 * amplitude
    assert abs(float(got - slope)) <= float(scale) * (HALF_STEP[dtype] + 1e-6)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_position_shapes_and_values(dtype):
    q, k = inputs(3, 40, 2, 1, 64, torch.float32, "bthd")
    inv_freq, _ = fused.rope_frequencies(64, 1e6, device=DEV)
    rows = torch.stack([torch.arange(40), 131071 - torch.arange(40), torch.full((40,), -5)]).to(DEV, dtype)
    one = rows[1]
    wide = rows.new_zeros(3, 80)[:, ::2].copy_(rows)  # positions with strides of their own
    for pos, want in ((rows, rows), (wide, rows), (one, one.expand(3, 40)), (one[None], one.expand(3, 40)),
                      (one.expand(3, 40), one.expand(3, 40))):
        qo, ko = fused.rope_at_positions(q, k, pos, inv_freq)
        theta = (want.double()[..., None] * inv_freq.double())[:, None]
        check(qo, q, theta, 1.0, 64, False)
        check(ko, k, theta, 1.0, 64, False)


def test_far_positions_keep_their_fraction_of_a_turn():
    q, k = inputs(1, 64, 2, 1, 64, torch.float32, "bhtd")
    inv_freq, _ = fused.rope_frequencies(64, 1e4, device=DEV)
    freq64 = inv_freq.double() * (1 + 1e-9)  # not on the fp32 grid
    for start in (10**6, 2**31 + 5, 2**33 + 1):
        pos = start + torch.arange(64, device=DEV)[None]
        qo, _ = fused.rope_at_positions(q, k, pos, freq64)
        check(qo, q, (pos.double()[..., None] * freq64)[:, None], 1.0, 64, False)


def test_one_side_only_and_empty_inputs():
    q, k = inputs(2, 8, 4, 2, 64, torch.bfloat16, "bthd")
    pos = torch.arange(8, device=DEV)
    inv_freq, _ = fused.rope_frequencies(32, device=DEV)
    qo, ko = fused.rope_at_positions(q, k, pos, inv_freq, interleaved=True)
    alone, none = fused.rope_at_positions(q, None, pos, inv_freq, interleaved=True)
    assert none is None and torch.equal(alone, qo)
    # only one of the outputs used, only one of the inputs a leaf
    q1, k1 = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    fused.rope_at_positions(q1, k1, pos, inv_freq, interleaved=True)[1].sum().backward()
    assert q1.grad is None and k1.grad is not None
    k2 = k.clone().requires_grad_(True)
    out = fused.rope_at_positions(q, k2, pos, inv_freq, interleaved=True)
    (out[0].sum() + out[1].sum()).backward()  # (the gradient of a sum is one number expanded)
    assert torch.equal(k2.grad, k1.grad)
    for shape in ((0, 4, 8, 64), (2, 4, 0, 64), (2, 0, 8, 64)):
        e = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        p = torch.arange(shape[2], device=DEV)
        a, b = fused.rope_at_positions(e, e, p, inv_freq)
        assert a.shape == shape and b.shape == shape


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("r", [32, 20])
def test_gradient_against_differences(r, interleaved):
    """The rotation is linear: the change of a weighted sum of its outputs along v is what its gradient says times v, for
    steps of any size.  Both sides are sums of terms whose values the kernel rounds as `check` counts."""
    q, k = inputs(2, 11, 3, 2, 32, torch.float32, "bthd", seed=5)
    v, _ = inputs(2, 11, 3, 2, 32, torch.float32, "bhtd", seed=6)
    g, _ = inputs(2, 11, 3, 2, 32, torch.float32, "bhtd", seed=7)
    inv_freq, _ = fused.rope_frequencies(r, device=DEV)
    pos = torch.arange(11, device=DEV) * 7
    f = lambda x: fused.rope_at_positions(x, k, pos, inv_freq, interleaved=interleaved, attention_scaling=1.25)[0]
    leaf = q.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(f(leaf), leaf, g)
    up, down = q + v, q - v
    step = (up.double() - down.double()) / 2  # what the rounded sums differ by
    change = ((f(up).double() - f(down).double()) / 2 * g.double()).sum()
    theta = torch.zeros((), device=DEV, dtype=torch.float64)
    size = lambda x: turned(x, theta, 1.25, r, interleaved)[1] * 1.25 + x.double().abs()
    part = 3.15 * 2.0**-25 + 2 * 2.0**-23 + 5 * 2.0**-24
    tol = part * ((size(up) + size(down)) / 2 * g.double().abs()).sum() + part * (size(g) * step.abs()).sum()
    assert abs(float(change - (dq.double() * step).sum())) <= float(tol)


def test_a_second_derivative_is_refused():
    q, k = inputs(1, 4, 1, 1, 8, torch.float32, "bhtd")
    q.requires_grad_(True)
    inv_freq, _ = fused.rope_frequencies(8, device=DEV)
    out, _ = fused.rope_at_positions(q, k, torch.arange(4, device=DEV), inv_freq)
    (g,) = torch.autograd.grad((out * out).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    q, k = inputs(2, 8, 4, 2, 64, torch.float32, "bhtd")
    pos, f = torch.arange(8, device=DEV), torch.ones(32, device=DEV)
    call = fused.rope_at_positions
    for bad in ((q, k[:1], pos, f), (q, k.bfloat16(), pos, f), (q.half(), None, pos, f), (q, k, pos[:7], f),
                (q, k, pos.float(), f), (q, k, pos, torch.ones(33, device=DEV)), (q, k, pos, f.bfloat16()),
                (q, k, pos, f[:0]), (q, k, pos, f[None]), (q[0], None, pos, f), (q, k, pos[None].expand(3, 8), f),
                (q, k, pos, torch.ones(32, device=DEV, requires_grad=True))):
        with pytest.raises(ValueError):
            call(*bad)
    with pytest.raises(RuntimeError):
        call(q, k, pos.cpu(), f)


def test_in_place_through_the_library():
    q, k = inputs(2, 19, 4, 2, 96, torch.bfloat16, "bthd")
    pos, (f, _) = torch.arange(19, device=DEV), fused.rope_frequencies(48, device=DEV)
    want = fused.rope_at_positions(q, k, pos, f)
    s = fused._strides6
    C.check(C.load().prl_rope_positions(q.data_ptr(), q.data_ptr(), s(q, q), 4, k.data_ptr(), k.data_ptr(), s(k, k), 2,
                                        pos.data_ptr(), 1, 0, 1, f.data_ptr(), 0, 48, 0, 1.0, C.PRL_BF16, 2, 19, 96, 0,
                                        C.stream_ptr(q.device)), "prl_rope_positions")
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_captured_and_replayed_and_on_other_streams():
    q, k = inputs(2, 130, 4, 2, 64, torch.bfloat16, "bthd")
    pos = torch.arange(260, device=DEV).view(2, 130)
    f, _ = fused.rope_frequencies(64, device=DEV)
    run = lambda: fused.rope_at_positions(q, k, pos, f, interleaved=True)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(3):
        q.normal_(), pos.add_(1000 * step)
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    with torch.cuda.stream(side):
        a = run()
    with torch.cuda.stream(other):
        b = run()
    torch.cuda.synchronize()
    assert torch.equal(a[0], want[0]) and torch.equal(b[0], want[0])


def test_heads_that_are_one_head_expanded():
    q, k = inputs(2, 21, 1, 1, 64, torch.bfloat16, "bthd")
    pos = torch.arange(21, device=DEV)
    f, _ = fused.rope_frequencies(64, device=DEV)
    k.requires_grad_(True)
    qo, ko = fused.rope_at_positions(q, k.expand(2, 6, 21, 64), pos, f)
    one = fused.rope_at_positions(q, k.detach(), pos, f)[1]
    assert torch.equal(ko, one.expand(2, 6, 21, 64))
    g = torch.randn(2, 6, 21, 64, device=DEV).bfloat16()
    ko.backward(g)  # the heads' gradients are added up
    theta = (pos.double()[:, None] * f.double())[None, None]
    want, m = turned(g, -theta, 1.0, 64, False)
    tol = (m * 6e-7 + 2.0**-8 * want.abs()).sum(1, keepdim=True) + 2.0**-8 * want.sum(1, keepdim=True).abs() + 6 * 2.0**-23
    assert bool(((k.grad.double() - want.sum(1, keepdim=True)).abs() <= tol).all())


def test_more_tokens_than_a_launch_has_workgroups_for():
    n = (1 << 23) + 12345  # two tokens a workgroup, 2^22 workgroups
    x = torch.randn(1, 1, n, 2, device=DEV)
    pos = torch.arange(n, device=DEV)
    f = torch.ones(1, device=DEV)
    out, _ = fused.rope_at_positions(x, None, pos, f)
    for cut in (slice(0, 1000), slice((1 << 23) - 1000, n)):
        check(out[:, :, cut], x[:, :, cut], pos[cut].double()[None, None, :, None], 1.0, 2, False)


def test_offsets_beyond_32_bits():
    t, heads, d = (1 << 17) + 3, 130, 128  # 2.2e9 elements
    x = torch.empty(1, t, heads, d, dtype=torch.bfloat16, device=DEV).normal_().transpose(1, 2)
    pos = torch.arange(t, device=DEV)
    inv_freq, _ = fused.rope_frequencies(d, device=DEV)
    out, _ = fused.rope_at_positions(x, None, pos, inv_freq)
    assert x.numel() > 2**31
    for cut in (slice(0, 5), slice(t // 2, t // 2 + 5), slice(t - 5, t)):
        alone, _ = fused.rope_at_positions(x[:, :, cut], None, pos[cut], inv_freq)
        assert torch.equal(out[:, :, cut], alone)
        check(alone, x[:, :, cut], pos[cut].double()[None, None, :, None] * inv_freq.double(), 1.0, d, False)
