"""The norms before and after a block with gate and residual scale, against the definition in 64 bits."""

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import _capi as C
from prime_rl_cse_amd import fused

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
U = 2.0**-24  # one fp32 rounding
E1, E2 = 1e-6, 1e-5


def make(rows, h, dtype, gate, post, pre, seed=0, lead=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=gen, device=DEV).to(dtype)
    lead = (rows,) if lead is None else lead
    shape = {None: None, "one": (), "channel": (h,), "token": (*lead, 1), "full": (*lead, h)}[gate]
    return {"x": mk(*lead, h) * 2, "b": mk(*lead, h), "w1": 1 + mk(h) * 0.25 if post else None,
            "w2": 1 + mk(h) * 0.25 if pre else None, "g": None if shape is None else mk(*shape),
            "gh": mk(*lead, h), "gy": mk(*lead, h) if pre else None}


def define(t, scale, offset):
    """(h, y) in float64, differentiable."""
    b = t["b"]
    n = b if t["w1"] is None else b * ((b * b).mean(-1, keepdim=True) + E1).rsqrt() * (t["w1"] + offset)
    h = t["x"] + scale * (n if t["g"] is None else t["g"] * n)
    y = None if t["w2"] is None else h * ((h * h).mean(-1, keepdim=True) + E2).rsqrt() * (t["w2"] + offset)
    return h, y


def bounds(t, scale, offset, rows):
    """Float64 values of every output, and for each the sum of the magnitudes of the terms it is made of."""
    d = {k: None if v is None else v.detach().double() for k, v in t.items()}
    width = d["x"].shape[-1]
    mean = lambda v: v.mean(-1, keepdim=True)
    w1 = torch.ones(width, dtype=torch.float64, device=DEV) if d["w1"] is None else d["w1"] + offset
    m1 = w1.abs() if d["w1"] is None else d["w1"].abs() + abs(offset)
    g = torch.ones((), dtype=torch.float64, device=DEV) if d["g"] is None else d["g"]
    r1 = 1.0 if d["w1"] is None else (mean(d["b"] ** 2) + E1).rsqrt()
    bh = d["b"] * r1
    n = bh * w1
    h = d["x"] + scale * g * n
    hm = d["x"].abs() + (scale * g * bh).abs() * m1
    want, mag = {"h": h}, {"h": hm}
    gh = d["gh"]
    G, Gm = gh, gh.abs()
    if d["w2"] is not None:
        w2, m2 = d["w2"] + offset, d["w2"].abs() + abs(offset)
        r2 = (mean(h * h) + E2).rsqrt()
        hh, hhm = h * r2, hm * r2
        q, qm = d["gy"] * w2, d["gy"].abs() * m2
        want["y"], mag["y"] = hh * w2, hhm * m2
        G = G + r2 * (q - hh * mean(q * hh))
        Gm = Gm + r2 * (qm + hhm * mean(qm * hhm))
        want["w2"], mag["w2"] = (d["gy"] * hh).flatten(0, -2).sum(0), (d["gy"].abs() * hhm).flatten(0, -2).sum(0)
    u, um = scale * g * G, (scale * g).abs() * Gm
    want["x"], mag["x"] = G, Gm
    q, qm = u * w1, um * m1
    if d["w1"] is None:
        want["b"], mag["b"] = q, qm
    else:
        want["b"] = r1 * (q - bh * mean(q * bh))
        mag["b"] = r1 * (qm + bh.abs() * mean(qm * bh.abs()))
        want["w1"], mag["w1"] = (u * bh).flatten(0, -2).sum(0), (um * bh.abs()).flatten(0, -2).sum(0)
    if d["g"] is not None:
        over = lambda v: v.sum_to_size(d["g"].shape)
        want["g"], mag["g"] = over(scale * G * n), over(abs(scale) * Gm * bh.abs() * m1)
    return want, mag


def check(t, scale=1.0, offset=0.0, train=True, **kw):
    leaves = {k: t[k].detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
              for k in ("x", "b", "w1", "w2", "g") if t[k] is not None}
    a = {**t, **leaves}
    h, y = fused.block_norms(a["x"], a["b"], a["w1"], a["w2"], gate=a["g"], scale=scale, eps=E1, pre_eps=E2,
                             weight_offset=offset)
    got = {"h": h, "y": y}
    if train:
        torch.autograd.backward([h] if y is None else [h, y], [t["gh"]] if y is None else [t["gh"], t["gy"]])
        got.update({k: leaves[k].grad for k in leaves})
    rows = h.numel() // max(1, h.shape[-1])
    want, mag = bounds(t, scale, offset, rows)
    for name in want:
        if name not in got:
            continue
        # Roundings along the longest chain to one element, each of at most U of the terms' magnitudes: a row's sum
        # (16 elements a thread, 6 steps over a wave, 16 waves) goes into r with half its relative error, rsqrt 2,
        # factors 6; the backward has two such sums after one another: 64 and 160.  Sums over rows: at most rows of a
        # workgroup in turn, then 4 + 32 + 32 partial sums.
        steps = 64 if name in "hy" else 160
        if name in ("w1", "w2", "g"):
            steps += 72 + rows // 256 + 1
        if name == "g" and t["g"].ndim == 0:  # the same again over a row: 16 elements a thread, 6 + 16
            steps += 38 * (1 + rows // 256)
        dt = t["x"].dtype
        tol = HALF_STEP[dt] * want[name].abs() * (1 + 2.0**-10) + steps * U * mag[name] + 1e-30
        err = (got[name].double() - want[name]).abs()
        assert got[name].dtype == dt and got[name].shape == want[name].shape, name
        assert bool((err <= tol).all()), (name, float((err / tol).max()))
    return got


CASES = [  # rows, h, gate, post, pre, scale, offset
    (1, 1, None, True, True, 1.0, 0.0),
    (1, 2048, None, True, True, 1.0, 0.0),
    (3, 8, "channel", True, True, 0.5, 1.0),
    (5, 7, "token", True, True, 1.0, 0.0),
    (37, 512, "full", True, True, 1.0, 0.0),
    (37, 520, "channel", True, True, 1.5, 1.0),
    (67, 1024, "token", True, True, 1.0, 0.0),
    (130, 1023, "channel", True, True, 1.0, 0.0),
    (9, 1531, "full", True, True, 0.25, 0.0),
    (300, 2056, "token", True, True, 1.0, 1.0),
    (11, 4097, "channel", True, True, 1.0, 0.0),
    (600, 5120, "channel", True, True, 1.0, 0.0),
    (7, 8192, "full", True, True, 1.0, 0.0),
    (7, 8191, "token", True, True, 1.0, 0.0),
    (2500, 264, "channel", True, True, 1.0, 0.0),
    (33, 896, None, False, True, 0.22, 0.0),
    (33, 3584, "channel", False, True, 0.22, 0.0),
    (33, 896, None, True, False, 1.0, 0.0),
    (33, 3584, "token", True, False, 1.0, 1.0),
    (33, 896, "full", False, False, 2.0, 0.0),
    (33, 2000, "channel", False, False, 2.0, 0.0),
    (12, 640, "one", True, True, 1.0, 0.0),
    (1500, 2000, "one", True, True, 1.0, 0.0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(case, dtype):
    rows, h, gate, post, pre, scale, offset = case
    t = make(rows, h, dtype, gate, post, pre)
    got = check(t, scale, offset)
    again = check(t, scale, offset)
    for k in got:  # same inputs, same bits
        assert got[k] is None or torch.equal(got[k], again[k])
    with torch.no_grad():  # the form without a backward
        hh, y = fused.block_norms(t["x"], t["b"], t["w1"], t["w2"], gate=t["g"], scale=scale, eps=E1, pre_eps=E2,
                                  weight_offset=offset)
    assert torch.equal(hh, got["h"]) and (y is None or torch.equal(y, got["y"]))


@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
def test_gradients_against_differences_of_the_definition(gate):
    t = make(6, 96, torch.float32, gate, True, True, seed=3)
    got = check(t, 0.7, 1.0)
    names = [k for k in ("x", "b", "w1", "w2", "g") if t[k] is not None]
    want, mag = bounds(t, 0.7, 1.0, 6)
    d = {k: None if v is None else v.double() for k, v in t.items()}
    f = lambda z: sum((o * w).sum() for o, w in zip(define(z, 0.7, 1.0), (d["gh"], d["gy"])))
    gen = torch.Generator(device=DEV).manual_seed(9)
    for k in names:
        v = torch.randn(t[k].shape, generator=gen, device=DEV, dtype=torch.float64)
        e = 1e-5
        slope = (f({**d, k: d[k] + e * v}) - f({**d, k: d[k] - e * v})) / (2 * e)
        err = abs(float((got[k].double() * v).sum() - slope))
        # the kernel's bound as above; central differences: e^2 of a third derivative of order one, and 1e-16 / e
        assert err <= float((mag[k] * v.abs()).sum()) * (260 * U + 1e-8), k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype):
    # three dimensions, rows inside wider rows, rows at an odd place
    t = make(0, 264, dtype, "token", True, True, lead=(3, 5))
    check(t)
    t = make(20, 264, dtype, "full", True, True)
    wide = torch.randn(20, 4, 264, device=DEV).to(dtype)
    t.update(x=wide[:, 0], b=wide[:, 1], g=wide[:, 2], gh=wide[:, 3])
    check(t)
    odd = torch.randn(4 * 20 * 267 + 1, device=DEV).to(dtype)[1:].view(4, 20, 267)[..., 2:266]
    t.update(x=odd[0], b=odd[1], g=odd[2], gy=odd[3])
    check(t)
    t.update(x=odd[0].t().contiguous().t())
    check(t)
    # a sum's gradient is one number expanded; an input that is one row expanded
    x = torch.randn(1, 64, device=DEV).to(dtype).requires_grad_(True)
    b = torch.randn(6, 64, device=DEV).to(dtype).requires_grad_(True)
    w = torch.ones(64, device=DEV, dtype=dtype)
    h, y = fused.block_norms(x.expand(6, 64), b, w, w)
    (h.sum() + y.sum()).backward()
    h2, y2 = fused.block_norms(x.detach().repeat(6, 1), b.detach(), w, w)
    assert torch.equal(h, h2) and torch.equal(y, y2) and x.grad.shape == (1, 64)


def test_outputs_that_go_nowhere():
    t = make(9, 200, torch.float32, "channel", True, True)
    for use in ("h", "y"):
        leaves = [t[k].clone().requires_grad_(True) for k in ("x", "b", "w1", "w2", "g")]
        h, y = fused.block_norms(*leaves[:4], gate=leaves[4], eps=E1, pre_eps=E2)
        (h * t["gh"] if use == "h" else y * t["gy"]).sum().backward()
        zero = torch.zeros_like(t["gh"])
        want, mag = bounds({**t, "gh": t["gh"] if use == "h" else zero, "gy": t["gy"] if use == "y" else zero}, 1.0, 0.0, 9)
        for k, leaf in zip(("x", "b", "w1", "w2", "g"), leaves):
            g = torch.zeros_like(leaf) if leaf.grad is None else leaf.grad
            assert bool(((g.double() - want[k]).abs() <= U * want[k].abs() + 260 * U * mag[k] + 1e-30).all()), (use, k)
        assert (leaves[3].grad is None) == (use == "h")


def test_empty_rows_and_zero_rows():
    w = torch.ones(48, device=DEV, requires_grad=True)
    x = torch.empty(0, 48, device=DEV, requires_grad=True)
    h, y = fused.block_norms(x, x, w, w, gate=torch.ones(48, device=DEV))
    (h.sum() + y.sum()).backward()
    assert h.shape == y.shape == (0, 48) and torch.equal(w.grad, torch.zeros(48, device=DEV))
    z = torch.zeros(3, 100, device=DEV)
    one = torch.ones(100, device=DEV)
    h, y = fused.block_norms(z, z, one, one)  # rsqrt(0 + eps) is finite: rows of zeros stay zeros
    assert torch.equal(h, z) and torch.equal(y, z)


@pytest.mark.parametrize("h", [100, 1000, 2001])
def test_infinities_and_nans_stay_in_their_row(h):
    t = make(8, h, torch.float32, "channel", True, True)
    clean = fused.block_norms(t["x"], t["b"], t["w1"], t["w2"], gate=t["g"])
    t["x"][2, 1], t["b"][5, h - 1] = float("inf"), float("nan")
    hid, y = fused.block_norms(t["x"], t["b"], t["w1"], t["w2"], gate=t["g"])
    want, wy = define({k: None if v is None else v.double() for k, v in t.items()}, 1.0, 0.0)
    for got, ref, was in ((hid, want, clean[0]), (y, wy, clean[1])):
        assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isinf(), ref.isinf())
        keep = [0, 1, 3, 4, 6, 7]
        assert torch.equal(got[keep], was[keep])


def test_refusals():
    x = torch.zeros(4, 16, device=DEV)
    w = torch.ones(16, device=DEV)
    call = fused.block_norms
    for bad in ((x, x[:3], w, w), (x, x.bfloat16(), w, w), (x, x, w.bfloat16(), w), (x, x, w[:8], w), (x.half(), x.half()),
                (torch.zeros(2, 8193, device=DEV), torch.zeros(2, 8193, device=DEV)),
                (torch.zeros(2, 0, device=DEV), torch.zeros(2, 0, device=DEV))):
        with pytest.raises(ValueError):
            call(*bad)
    for gate in (torch.ones(3, 1, device=DEV), torch.ones(1, 16, device=DEV), torch.ones(15, device=DEV), torch.ones(4, 16, device=DEV).bfloat16()):
        with pytest.raises(ValueError):
            call(x, x, w, w, gate=gate)
    with pytest.raises(RuntimeError):
        call(x, x.cpu(), w, w)


def test_captured_with_its_backward_and_replayed():
    t = make(70, 1032, torch.bfloat16, "channel", True, True)
    leaves = [t[k].clone().requires_grad_(True) for k in ("x", "b", "w1", "w2", "g")]

    def run():
        out = fused.block_norms(*leaves[:4], gate=leaves[4])
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, [t["gh"], t["gy"]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs that know nothing of one another
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for _ in range(3):
        with torch.no_grad():
            leaves[0].normal_(), leaves[1].normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = run()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    a, b = (make(500, 2048, torch.bfloat16, "full", True, True, seed=s) for s in (1, 2))
    want = [check(t) for t in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(4):
        for i, (t, s) in enumerate(zip((a, b), streams)):
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                leaves = [t[k].clone().requires_grad_(True) for k in ("x", "b", "w1", "w2", "g")]
                out = fused.block_norms(*leaves[:4], gate=leaves[4], eps=E1, pre_eps=E2)
                outs[i].append(torch.autograd.grad(out, leaves, [t["gh"], t["gy"]]))
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        for g in got:
            assert all(torch.equal(v, ref[k]) for v, k in zip(g, ("x", "b", "w1", "w2", "g")))


def test_library_leaves_what_lies_between_rows():
    rows, h = 6, 200
    t = make(rows, h, torch.bfloat16, None, True, True)
    out = torch.full((2, rows, h + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    C.check(C.load().prl_block_norms_fwd(
        t["x"].data_ptr(), h, t["b"].data_ptr(), h, t["w1"].data_ptr(), t["w2"].data_ptr(), C.GATE_NONE, None, 0, 1.0, 0.0,
        E1, E2, out[0].data_ptr(), h + 24, out[1].data_ptr(), h + 24, None, None, C.PRL_BF16, rows, h,
        C.stream_ptr(out.device)), "prl_block_norms_fwd")
    hid, y = fused.block_norms(t["x"], t["b"], t["w1"], t["w2"], eps=E1, pre_eps=E2)
    assert torch.equal(out[0, :, :h], hid) and torch.equal(out[1, :, :h], y) and bool((out[..., h:] == 7).all())


@pytest.mark.parametrize("rows, h", [((1 << 20) + 33, 2056), ((1 << 22) + 9, 8)])  # 2.2e9 elements; more rows than waves
def test_many_rows(rows, h):
    """Far rows come out as they do by themselves, bit for bit, both ways."""
    mk = lambda: torch.empty(rows, h, dtype=torch.bfloat16, device=DEV).normal_()
    x, b, gh, gy = mk().requires_grad_(True), mk().requires_grad_(True), mk(), mk()
    w = torch.rand(h, device=DEV).to(torch.bfloat16)
    run = lambda x, b: fused.block_norms(x, b, w, w, scale=0.5, eps=E1, pre_eps=E2)
    out = run(x, b)
    grads = torch.autograd.grad(out, [x, b], [gh, gy])
    for cut in (slice(0, 7), slice(rows // 2, rows // 2 + 7), slice(rows - 7, rows)):
        xs, bs = (v.detach()[cut].clone().requires_grad_(True) for v in (x, b))
        alone = run(xs, bs)
        for got, want in zip((*out, *grads), (*alone, *torch.autograd.grad(alone, [xs, bs], [gh[cut], gy[cut]]))):
            assert torch.equal(got[cut], want)
