"""Calls at the edges of the fused layers' host side: norms whose instances differ, tables, hooks, gradients that share
memory.  Host only; the kernels' side is tests/test_gpu_operator_edges.py."""

import copy

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import fused


@pytest.fixture(autouse=True)
def one_thread():
    """Tiny tensors: handing them to threads takes longer than the work."""
    threads = torch.get_num_threads()
    torch.set_num_threads(1)
    yield
    torch.set_num_threads(threads)


class FlaggedNorm(torch.nn.Module):
    """An RMSNorm whose instances say for themselves whether the weight is a distance from one."""

    def __init__(self, from_one, width=8):
        super().__init__()
        self.eps, self.from_one = 1e-6, from_one
        self.weight = torch.nn.Parameter(torch.rand(width))

    def forward(self, x):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.eps)
        return y * (1.0 + self.weight if self.from_one else self.weight)


@pytest.mark.parametrize("order", [(False, True), (True, False)])
def test_a_norm_s_form_belongs_to_the_instance(order):
    norms = [FlaggedNorm(flag) for flag in order]
    for _ in range(2):  # (asked again: what was found is kept on the module)
        assert [fused._norm_form(n) for n in norms] == [float(flag) for flag in order]


def test_a_norm_whose_forward_was_replaced_has_no_form():
    norm = FlaggedNorm(False)
    norm.forward = lambda x: x * 2
    assert fused._norm_form(norm) is None


def test_a_norm_that_uses_another_epsilon_has_no_form():
    class Norm(FlaggedNorm):
        def forward(self, x):
            return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1.5e-6) * self.weight

    assert fused._norm_form(Norm(False)) is None


def test_a_norm_s_form_is_found_under_other_defaults():
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.bfloat16)
        assert fused._norm_form(FlaggedNorm(True)) == 1.0
    finally:
        torch.set_default_dtype(before)


def test_fuse_model_asks_norms_anew():
    norm = FlaggedNorm(False)
    assert fused._norm_form(norm) == 0.0
    other = copy.deepcopy(norm)
    other.from_one = True
    fused.fuse_model(torch.nn.ModuleList([other]))
    assert fused._norm_form(other) == 1.0 and fused._norm_form(norm) == 0.0


@pytest.mark.parametrize("post", [False, True])
def test_a_norm_of_unknown_form_is_called(post, monkeypatch):
    """One norm alone, and it is none the kernel knows: step by step."""
    monkeypatch.setattr(fused, "block_norms_supported", lambda *a, **k: True)
    norm = torch.nn.LayerNorm(8)
    x, branch = torch.randn(3, 8), torch.randn(3, 8)
    hidden, normed = fused._between_blocks(x, branch, norm if post else None, 0.5, None if post else norm)
    want = x + 0.5 * (norm(branch) if post else branch)
    assert torch.equal(hidden, want) and torch.equal(normed, want if post else norm(want))


def sandwich(name="Glm4"):
    from tests.test_fuse_families import tiny

    model = tiny(name, num_hidden_layers=2)
    gen = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn(p.shape, generator=gen) * 0.05)
    return model


def stepwise(monkeypatch):
    """`block_norms` and `add_rms_norm` from elementary operations, so that the fused layers run on the host."""
    rms = lambda v, w, eps: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * w
    calls = []

    def block_norms(x, branch, w1, w2, *, scale, eps, pre_eps, weight_offset):
        calls.append("block_norms")
        hidden = x + scale * (branch if w1 is None else rms(branch, w1 + weight_offset, eps))
        return hidden, None if w2 is None else rms(hidden, w2 + weight_offset, pre_eps)

    def add_rms_norm(x, branch, w, eps):
        calls.append("add_rms_norm")
        return x + branch, rms(x + branch, w, eps)

    monkeypatch.setattr(fused, "block_norms_supported", lambda *a, **k: True)
    monkeypatch.setattr(fused, "block_norms", block_norms)
    monkeypatch.setattr(fused, "add_rms_norm_supported", lambda *a: True)
    monkeypatch.setattr(fused, "add_rms_norm", add_rms_norm)
    return calls


def logits(model):
    ids = torch.arange(2 * 12).view(2, 12) % 160
    return model(input_ids=ids, position_ids=torch.arange(12).expand(2, 12)).logits


def close(a, b):  # fp32, two layers: a norm left out or a hook not run changes values by their own size
    return bool((a - b).abs().max() <= 2000 * 2.0**-24 * b.abs().max())


HOOKS = {
    "forward": lambda m: m.register_forward_hook(lambda mod, args, out: out * 1.5),
    "pre": lambda m: m.register_forward_pre_hook(lambda mod, args: (args[0] * 0.5 + 1.0,)),
    "global": lambda m: torch.nn.modules.module.register_module_forward_hook(
        lambda mod, args, out: out * 1.5 if mod is m else None),
}


@pytest.mark.parametrize("carry", [False, True])
@pytest.mark.parametrize("kind", list(HOOKS))
@pytest.mark.parametrize("name", ["Glm4", "Gemma2", "Olmo2", "Granite", "Qwen3"])
def test_hooks_on_norms_run(name, kind, carry, monkeypatch):
    model = sandwich(name)
    norms = {n: m for n, m in model.named_modules() if n.startswith("model.") and type(m).__name__.endswith("RMSNorm")
             and "self_attn" not in n}
    stepwise(monkeypatch)
    for n, m in norms.items():
        handle = HOOKS[kind](m)
        try:
            want = logits(model)
            fused.fuse_model(model)
            try:
                fused.enable_residual_carry(model, carry)
                assert close(logits(model), want), n
            finally:
                fused.unfuse_model(model)
        finally:
            handle.remove()
        assert not close(logits(model), want), n  # (the hook did change something)


@pytest.mark.parametrize("name", ["Glm4", "Granite", "Qwen3"])
def test_hooks_on_layers_see_whole_hidden_states(name, monkeypatch):
    model = sandwich(name)
    calls = stepwise(monkeypatch)

    def look():
        seen = []
        handles = []
        for m in (*model.model.layers, model.model.norm):
            handles.append(m.register_forward_pre_hook(lambda mod, args: seen.append(args[0].detach().clone())))
            handles.append(m.register_forward_hook(lambda mod, args, out: seen.append(out.detach().clone())))
        logits(model)
        for h in handles:
            h.remove()
        return seen

    want = look()
    fused.fuse_model(model)
    try:
        assert fused.enable_residual_carry(model) == 2
        got = look()
        assert len(got) == len(want) == 6 and all(close(a, b) for a, b in zip(got, want))
        # one layer's hook alone leaves the others their carry; a hook that looks at nothing leaves it to all
        plain = logits(model)
        calls.clear()
        logits(model)
        every = list(calls)
        hook = lambda mod, args: None
        hook.looks_at_nothing = True
        handle = model.model.layers[1].register_forward_pre_hook(hook)
        calls.clear()
        assert torch.equal(logits(model), plain) and calls == every
        handle.remove()
    finally:
        fused.unfuse_model(model)
    assert not hasattr(model.model.layers[0], "_prl_at")


def test_backward_hooks_on_norms_run(monkeypatch):
    model = sandwich("Glm4")
    stepwise(monkeypatch)
    fused.fuse_model(model)
    try:
        seen = []
        for layer in model.model.layers:
            layer.post_mlp_layernorm.register_full_backward_hook(lambda mod, gi, go: seen.append(tuple(go[0].shape)))
        logits(model).sum().backward()
        assert seen == [(2, 12, 64)] * 2
    finally:
        fused.unfuse_model(model)


def test_fuse_model_leaves_norms_that_add_one_to_their_weight():
    class FlaggedRMSNorm(FlaggedNorm):
        def __init__(self, from_one):
            super().__init__(from_one)
            self.variance_epsilon = self.eps

    norms = torch.nn.ModuleList([FlaggedRMSNorm(False), FlaggedRMSNorm(True)])
    assert fused.fuse_model(norms)["rmsnorm"] == 1
    assert hasattr(norms[0], "_prl_torch_forward") and not hasattr(norms[1], "_prl_torch_forward")


def test_a_plain_layer_with_norms_that_add_one_is_left_alone():
    plain, layer = sandwich("Qwen3").model.layers
    assert fused._is_plain_decoder_layer(plain)

    class FromOneRMSNorm(type(layer.input_layernorm)):
        def forward(self, x):
            return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.variance_epsilon) * (1.0 + self.weight)

    layer.post_attention_layernorm.__class__ = FromOneRMSNorm
    assert not fused._is_plain_decoder_layer(layer)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad, monkeypatch):
    """Neither operator has one: a call on dual tensors fails instead of dropping the tangents."""
    import torch.autograd.forward_ad as fa

    monkeypatch.setattr(fused, "block_norms_supported", lambda *a: True)
    monkeypatch.setattr(fused, "_launch_block_norms", lambda *a: None)
    monkeypatch.setattr(fused, "rope_at_positions_supported", lambda *a: True)
    monkeypatch.setattr(fused, "_launch_rope_positions", lambda q, k, *a: (q.clone(), None if k is None else k.clone()))
    x, w, gate = torch.randn(3, 8), torch.randn(8), torch.rand(3, 1)
    q, pos, freq = torch.randn(1, 2, 3, 8), torch.arange(3), torch.ones(4)
    norms = lambda *t: fused.block_norms(*t[:4], gate=t[4])
    rope = lambda *t: fused.rope_at_positions(*t, pos, freq)
    with torch.set_grad_enabled(grad), fa.dual_level():
        for call, args in ((norms, [x, x.clone(), w, w.clone(), gate]), (rope, [q, q.clone()])):
            for i, t in enumerate(args):
                dual = list(args)
                dual[i] = fa.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError):
                    call(*dual)
            call(*args)  # (a level that none of the inputs takes part in)
        rope(q, None)


WINDOWS = [(1, 1), (0, 1), (3, 1), (8, 1), (12, 1), (1, 0), (2, 3)]  # strides of 5 rows of 8 out of one run of memory


@pytest.mark.parametrize("strides", WINDOWS)
def test_outputs_of_overlapping_rows_lie_row_by_row(strides, monkeypatch):
    """Inputs that are windows of one run of memory: the kernels write rows of their own pitch."""
    seen = []

    def run(fn, name, dev, *args):
        seen.append(name)

    monkeypatch.setattr(fused.C, "run", run)
    monkeypatch.setattr(fused.C, "stream_ptr", lambda dev: 0)
    monkeypatch.setattr(fused, "block_norms_supported", lambda *a: True)
    base = torch.randn(100)
    x, b = (base[i:].as_strided((5, 8), strides) for i in (0, 1))
    w = torch.ones(8)
    for t in fused.block_norms(x, b, w, w):
        assert t.stride() == (8, 1)
    out = fused.block_norms(x.requires_grad_(True), b, w, w)
    for t in (*out, *torch.autograd.grad(out, [x], [torch.ones(5, 8)] * 2)):
        assert t.stride() == (8, 1)
    assert seen == ["prl_block_norms_fwd"] * 2 + ["prl_block_norms_bwd"]


@pytest.mark.parametrize("strides", [(60, 30, 1, 1), (0, 1, 0, 1), (1, 40, 8, 1), (0, 0, 0, 1), (1, 1, 1, 1), (80, 8, 16, 1),
                                     (90, 40, 8, 0), (90, 45, 9, 1)])
def test_rotated_heads_of_overlapping_memory_lie_along_the_head(strides, monkeypatch):
    monkeypatch.setattr(fused.C, "run", lambda *a: None)
    monkeypatch.setattr(fused.C, "stream_ptr", lambda dev: 0)
    q = torch.randn(400).as_strided((3, 2, 5, 8), strides)
    for inverse in (False, True):
        qo, ko = fused._launch_rope_positions(q, q, torch.arange(5)[None], torch.ones(4), False, 1.0, inverse)
        for t in (qo, ko):
            assert t.stride(3) == 1
            span = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            assert span == t.numel() and t.untyped_storage().nbytes() >= 4 * span  # dense: no two elements in one place
    dense = torch.randn(3, 5, 2, 8).transpose(1, 2)
    assert fused._launch_rope_positions(dense, None, torch.arange(5)[None], torch.ones(4), False, 1.0, False)[0].stride() == \
        dense.stride()  # layouts of dense inputs are kept


def on_device(monkeypatch):
    """Host gradients pass for a device's, so that what is said about their memory can be asked here."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)


def test_gradients_that_share_memory_are_not_supported(monkeypatch):
    from prime_rl_cse_amd import optim

    on_device(monkeypatch)
    flat = torch.randn(40)
    apart = [flat[:10], flat[10:20], flat[25:], torch.randn(3).bfloat16(), flat[5:5]]
    assert optim.clip_grad_norm_supported(apart) and optim.clip_grad_norm_supported([])
    for shared in ([flat[:10], flat[9:12]], [flat, flat], [*apart, flat[12:13]], [flat[8:12], *apart]):
        assert not optim.clip_grad_norm_supported(shared)
        with pytest.raises(ValueError):
            optim._pieces(shared, True)


@pytest.mark.parametrize("shared", [False, True])
def test_a_step_with_gradients_that_share_memory_clips_by_torch(shared, monkeypatch):
    """`train_step` hands to the package's clipping only what that takes."""
    from prime_rl_cse_amd import trainer as T

    on_device(monkeypatch)
    flat = torch.randn(12)
    params = [torch.nn.Parameter(torch.zeros(4)) for _ in range(2)]
    params[0].grad, params[1].grad = flat[:4], (flat[3:7] if shared else flat[4:8])
    taken = []
    monkeypatch.setattr(T, "clip_grad_norm_", lambda p, m: taken.append("package") or torch.tensor(1.0))
    monkeypatch.setattr(torch.nn.utils, "clip_grad_norm_", lambda p, m: taken.append("torch") or torch.tensor(1.0))
    T._clip(params, 1.0)
    assert taken == ["torch" if shared else "package"]


def test_no_rows_and_no_gate_is_refused():
    """The sums over no rows are still formed by a launch, which reads a gate per channel once."""
    from prime_rl_cse_amd import _capi as C

    lib, one, none = C.load(), 16, None
    bwd = lambda rows: lib.prl_block_norms_bwd(one, 16, one, 16, one, one, C.GATE_CHANNEL, none, 16, 1.0, 0.0, one, one, none,
                                               0, one, 16, one, 16, one, 16, one, one, none, 16, 0, rows, 16, one, 1 << 20,
                                               none)
    assert bwd(2) == -1 and bwd(0) == -1
    # without a row and without a launch no gate is read
    assert lib.prl_block_norms_fwd(one, 16, one, 16, one, one, C.GATE_CHANNEL, none, 0, 1.0, 0.0, 1e-6, 1e-6, one, 16, one, 16,
                                   none, none, 0, 0, 16, none) == 0


def test_a_learned_factor_on_the_residual_leaves_the_layer_alone():
    """The kernel's factor is a number: a tensor's gradient would be lost."""
    layer = sandwich("Granite").model.layers[0]
    assert fused._layer_steps(layer) is not None
    layer.residual_multiplier = torch.nn.Parameter(torch.tensor(0.5))
    assert fused._layer_steps(layer) is None
    layer = sandwich("Granite").model.layers[0]
    layer.residual_multiplier = torch.tensor(0.5)
    assert fused._layer_steps(layer) is None


class OtherRotaryEmbedding(torch.nn.Module):
    """Tables of another kind, from a length: what a vision tower keeps beside the decoder's."""

    def __init__(self):
        super().__init__()
        self.register_buffer("inv_freq", torch.rand(4))

    def forward(self, length):
        return torch.outer(torch.arange(length), self.inv_freq)


@pytest.mark.parametrize("first", [False, True])
def test_only_rotary_modules_that_do_what_was_found_are_tagged(first):
    """Each module is tried by itself: another one in the model keeps its own forward."""
    import sys

    model = sandwich("Glm4")
    rotary, other = model.model.rotary_emb, OtherRotaryEmbedding()
    doubled = copy.deepcopy(rotary)  # the same class, another relation between tables and frequencies
    doubled.register_buffer("inv_freq", rotary.inv_freq.clone())
    doubled.forward = lambda x, pos: tuple(2 * t for t in type(rotary).forward(doubled, x, pos))
    extra = torch.nn.ModuleList([other, doubled])
    if first:
        model._modules = {"extra": extra, **model._modules}
    else:
        model.extra = extra
    kind, tagged = fused._rope_kind(sys.modules[type(model).__module__], model)
    assert kind == "interleaved" and tagged == [rotary]
    fused.fuse_model(model)
    try:
        assert other(3).shape == (3, 4)
        cos, _ = doubled(torch.zeros(1, 1, 3, 16), torch.arange(3)[None])
        assert not hasattr(cos, "_prl_rope")
        assert hasattr(rotary(torch.zeros(1, 1, 3, 16), torch.arange(3)[None])[0], "_prl_rope")
    finally:
        fused.unfuse_model(model)


def test_pairs_are_found_under_other_defaults():
    import sys

    model = sandwich("Glm4")
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.bfloat16)
        kind, tagged = fused._rope_kind(sys.modules[type(model).__module__], model)
    finally:
        torch.set_default_dtype(before)
    assert kind == "interleaved" and tagged == [model.model.rotary_emb]


def rotated_by(monkeypatch, kind="interleaved"):
    taken = []
    monkeypatch.setattr(fused, "rope_at_positions_supported", lambda *a: True)
    monkeypatch.setattr(fused, "rope_at_positions", lambda q, k, *a, **kw: taken.append("positions") or (q, k))
    return taken, fused._family_rope(lambda q, k, cos, sin, *a, **kw: taken.append("tables") or (q, k), kind)


def tables(model=None, dtype=torch.float32, t=5):
    rotary = (model or sandwich("Glm4")).model.rotary_emb
    rotary._prl_torch_forward = rotary.forward
    return fused._tagged_rotary_forward(rotary, torch.zeros(1, 2, t, 16, dtype=dtype), torch.arange(t)[None])


@pytest.mark.parametrize("extra", [(torch.arange(5)[None],), (2,), (None,), (1.0,), (True,), (2, 1)])
def test_other_arguments_go_to_the_family_s_function(extra, monkeypatch):
    """Positions behind the tables, another axis for the heads: only the plain call is taken over."""
    taken, rotate = rotated_by(monkeypatch)
    cos, sin = tables()
    q = torch.randn(1, 2, 5, 16)
    rotate(q, q, cos, sin, *extra)
    rotate(q, q, cos, sin, unsqueeze_dim=extra[0])
    rotate(q, q, cos, sin, position_ids=extra[0])
    assert taken == ["tables"] * 3
    taken.clear()
    rotate(q, q, cos, sin), rotate(q, q, cos, sin, 1), rotate(q, q, cos, sin, unsqueeze_dim=1)
    assert taken == ["positions"] * 3


def test_tables_of_another_type_go_to_the_family_s_function(monkeypatch):
    """Under autocast query and key are narrower than the tables; the family's function returns the wider type then."""
    taken, rotate = rotated_by(monkeypatch)
    cos, sin = tables()
    rotate(*[torch.randn(1, 2, 5, 16).bfloat16()] * 2, cos, sin)
    rotate(*[torch.randn(1, 2, 5, 16)] * 2, cos, sin)
    assert taken == ["tables", "positions"]


class SpreadOut(torch.Tensor):
    """A device tensor whose elements lie somewhere else (as a DTensor's do), as far as the checks can see."""

    is_cuda = property(lambda self: True)

    def to_local(self):
        raise AssertionError


def test_distributed_tensors_are_not_supported():
    x, w = torch.randn(3, 8), torch.ones(8)
    far = lambda t: t.as_subclass(SpreadOut)
    assert not fused.block_norms_supported(far(x), x, w, w)
    q, pos, freq = torch.randn(1, 2, 5, 8), torch.arange(5), torch.ones(4)
    assert not fused.rope_at_positions_supported(far(q), None, pos, freq)
    near = torch.randn(1, 2, 5, 8).as_subclass(type("Near", (torch.Tensor,), {"is_cuda": SpreadOut.is_cuda}))
    assert fused.rope_at_positions_supported(near, None, pos, freq)
    for args in ((near, far(q), pos, freq), (near, None, far(pos), freq), (near, None, pos, far(freq))):
        assert not fused.rope_at_positions_supported(*args)


def test_what_the_rotary_entry_refuses_is_not_supported():
    device = type("Near", (torch.Tensor,), {"is_cuda": SpreadOut.is_cuda})
    far = lambda *shape: torch.empty(1).expand(shape).as_subclass(device)
    ok = fused.rope_at_positions_supported
    pos, freq = torch.arange(3), torch.ones(4)
    assert ok(far(1, 2, 3, 1 << 20), None, pos, freq) and not ok(far(1, 2, 3, (1 << 20) + 2), None, pos, freq)
    assert ok(far(1, (1 << 19), 3, 8), far(1, (1 << 19) - 1, 3, 8), pos, freq)
    assert not ok(far(1, 1 << 19, 3, 8), far(1, 1 << 19, 3, 8), pos, freq)
    assert not ok(far(1, 1 << 20, 3, 8), None, pos, freq)
    assert ok(far(0, 2, 3, 8), None, pos, freq)


def host_clip(monkeypatch):
    """`clip_grad_norm_` and `grad_norm` up to their launches."""
    from prime_rl_cse_amd import _capi as C
    from prime_rl_cse_amd import optim

    on_device(monkeypatch)
    tables = []
    monkeypatch.setattr(optim, "_one_device", lambda parts: parts[0].device)
    monkeypatch.setattr(C, "run", lambda fn, name, dev, *a: tables.append(name))
    monkeypatch.setattr(C, "stream_ptr", lambda dev: 0)
    monkeypatch.setattr(C, "check", lambda code, name: None)
    monkeypatch.setattr(optim, "_norm_and_factor", lambda table, *a: tables.append(table.copy()) or torch.ones(2))

    class Lib:
        prl_grad_clip = None
        prl_grad_scale = staticmethod(lambda *a: 0)
        prl_grad_norm_workspace_bytes = staticmethod(lambda at, n: 8)

    monkeypatch.setattr(C, "load", lambda: Lib)
    return optim, tables


@pytest.mark.parametrize("shape", [(), (7,), (4, 5), (2, 3, 4)])
def test_the_norm_of_one_tensor(shape, monkeypatch):
    optim, tables = host_clip(monkeypatch)
    t = torch.randn(shape)
    optim.grad_norm(t)
    optim.grad_norm(t.t() if t.ndim == 2 else t)
    assert [(int(p["x"]), int(p["n"])) for table in tables for p in table] == [(t.data_ptr(), t.numel())] * 2


@pytest.mark.parametrize("check", [False, True])
def test_clipping_counts_as_a_write(check, monkeypatch):
    """A graph that has kept a gradient refuses its backward after the gradient was scaled, as after torch's own clipping."""
    optim, _ = host_clip(monkeypatch)
    params = [torch.nn.Parameter(torch.zeros(4)) for _ in range(3)]
    for p in params[:2]:
        p.grad = torch.randn(4)
    w = torch.ones(4, requires_grad=True)
    kept = (params[1].grad * w).sum()
    optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=check)
    assert [p.grad._version for p in params[:2]] == [1, 1]
    with pytest.raises(RuntimeError):
        kept.backward()
    with torch.inference_mode():  # (tensors that count no writes)
        quiet = torch.nn.Parameter(torch.zeros(4))
        quiet.grad = torch.randn(4)
        optim.clip_grad_norm_([quiet, params[0]], 1.0, error_if_nonfinite=check)
    assert params[0].grad._version == 2


@pytest.mark.parametrize("both", [False, True])
def test_a_rotary_module_that_cannot_be_copied_is_left_alone(both):
    import sys

    model = sandwich("Glm4")
    rotary = model.model.rotary_emb
    if not both:
        model.extra = copy.deepcopy(rotary)
    rotary.open_file = (i for i in range(2))
    home = sys.modules[type(model).__module__]
    found = fused._rope_kind(home, model)
    assert found is None if both else found == ("interleaved", [model.extra])
    try:
        fused.fuse_model(model)
    finally:
        fused.unfuse_model(model)


def test_a_deep_model_that_carries_can_be_copied():
    class Inner(torch.nn.Module):
        def __init__(self, layers, norm):
            super().__init__()
            self.layers, self.norm = torch.nn.ModuleList(layers), norm

    model = torch.nn.Module()
    base = sandwich("Qwen3").model
    model.model = Inner([copy.deepcopy(base.layers[0]) for _ in range(300)], base.norm)
    fused.fuse_model(model)
    assert fused.enable_residual_carry(model) == 300
    other = copy.deepcopy(model)
    first, last = other.model.layers[0], other.model.layers[-1]
    assert first._prl_carry is last._prl_carry is other.model.norm._prl_carry is not model.model.norm._prl_carry
    assert fused._hands_on(first) and fused._hands_on(last)
    other.model.norm.register_forward_hook(lambda *a: None)
    assert fused._hands_on(first) and not fused._hands_on(last) and fused._hands_on(model.model.layers[-1])


def test_hooks_that_wait_for_weights_leave_the_carry(monkeypatch):
    """The exchange's own pre-hooks (`Replica`): on layers, the final norm, and norms by themselves."""
    from types import SimpleNamespace

    from prime_rl_cse_amd.replica import Replica

    model = sandwich("Glm4")
    calls = stepwise(monkeypatch)
    fused.fuse_model(model)
    try:
        fused.enable_residual_carry(model)
        want = logits(model)
        expected = list(calls)
        params = list(model.parameters())
        inside = {id(p) for p in model.model.layers[1].parameters()}
        names = {id(p): n for n, p in model.named_parameters()}
        # the second layer cut: its norms in a bucket of their own, so that they get hooks of their own
        bucket_of = [2 if id(p) in inside and "layernorm" in names[id(p)] else 1 if id(p) in inside else 0 for p in params]
        waited = []
        state = SimpleNamespace(params=params, bucket_of=bucket_of, buckets=[0, 1, 2], wait_gathered=waited.append)
        Replica._hook_weight_arrival(SimpleNamespace(model=model, state=state))
        assert all(fused._hands_on(m) for m in model.model.layers)
        calls.clear()
        assert close(logits(model), want)
        # each of the cut layer's four norms was waited for (called as a module where it has its own hook)
        assert waited.count(2) == 4 and len(calls) < len(expected)
    finally:
        fused.unfuse_model(model)


def attention_blocks_taken(model, monkeypatch):
    """How many attention blocks of one forward the fused form asks for their stacked projection."""
    asked = []
    monkeypatch.setattr(fused, "_stackable", lambda x, *linears: asked.append(len(linears)))
    model(input_ids=torch.arange(12)[None], position_ids=torch.arange(12)[None])
    return asked.count(3) - len(model.model.layers)  # (the query projection of a block that runs by itself asks once)


def wide_heads():
    from tests.test_fuse_families import tiny

    return tiny("Qwen3", head_dim=128, num_attention_heads=2, num_key_value_heads=1)


def test_a_query_norm_that_adds_one_keeps_the_attention_block_s_own_forward(monkeypatch):
    model = wide_heads()

    class FromOneRMSNorm(type(model.model.norm)):
        def forward(self, x):
            return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.variance_epsilon) * (1.0 + self.weight)

    model.model.layers[0].self_attn.k_norm.__class__ = FromOneRMSNorm
    fused.fuse_model(model)
    try:
        assert [hasattr(m.self_attn, "_prl_torch_forward") for m in model.model.layers] == [False, True]
    finally:
        fused.unfuse_model(model)


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
def test_an_attention_block_with_hooks_on_its_norms_runs_its_own_forward(which, monkeypatch):
    model = wide_heads()
    fused.fuse_model(model)
    try:
        assert attention_blocks_taken(model, monkeypatch) == 2
        seen = []
        getattr(model.model.layers[1].self_attn, which).register_forward_hook(lambda *a: seen.append(1))
        assert attention_blocks_taken(model, monkeypatch) == 1 and len(seen) == 1
    finally:
        fused.unfuse_model(model)
