"""Model families whose layers are not of the plain shape (norms behind the blocks, factors on the residual, part of a
head rotated, neighbouring pairs) through `fuse_model`, and one whole optimizer step of such a model."""

import copy

import pytest
import torch

import prime_rl_cse_amd as prl
from prime_rl_cse_amd import fused
from prime_rl_cse_amd import trainer as T
from tests.test_fuse_families import tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(model, ids, pos, weights):
    model.zero_grad(set_to_none=True)
    logits = T.forward(model, ids, pos)
    (logits.float() * weights).sum().backward()
    return logits.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


# launches of one forward and backward of two layers: rotary from positions, norms around a block
FAMILIES = {"Glm4": (4, 4), "Gemma2": (0, 4), "Olmo2": (0, 4), "Granite": (0, 4), "Helium": (4, 0), "Cohere": (4, 0),
            "Glm4Moe": (4, 0)}


@pytest.mark.parametrize("name", list(FAMILIES))
def test_logits_and_gradients_are_those_of_the_unfused_model(name):
    model = tiny(name, **({"residual_multiplier": 0.22} if name == "Granite" else {})).to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(3)
    with torch.no_grad():
        for p in model.parameters():  # norm weights away from one
            p.add_(torch.randn(p.shape, generator=gen, device=DEV) * 0.05)
    ids = torch.randint(0, 160, (2, 48), generator=gen, device=DEV)
    pos = torch.arange(48, device=DEV).expand(2, 48)
    weights = torch.randn(2, 48, 160, generator=gen, device=DEV)
    want, wgrads = run(model, ids, pos, weights)
    fused.fuse_model(model)
    timer = prl._capi.KernelTimer()
    prl._capi.set_timer(timer)
    try:
        got, grads = run(model, ids, pos, weights)
    finally:
        prl._capi.set_timer(None)
        fused.unfuse_model(model)
    seen = timer.summary()
    count = lambda *names: sum(seen[n]["launches"] for n in names if n in seen)
    assert (count("prl_rope_positions"), count("prl_block_norms_fwd")) == FAMILIES[name]
    assert count("prl_block_norms_bwd") == FAMILIES[name][1]
    # fp32 on both sides: a few thousand roundings deep, 2^-24 each of the values' size; a pair taken wrong or a norm left
    # out changes them by the values' size itself
    assert (got - want).abs().max() <= 2000 * 2.0**-24 * want.abs().max()
    for n, g in grads.items():
        ref = wgrads[n]
        assert (g - ref).norm() <= 2000 * 2.0**-24 * ref.norm() + 1e-12, n
    again, _ = run(model, ids, pos, weights)
    assert torch.equal(again, want)  # everything is as it was


@pytest.mark.parametrize("name", ["Glm4", "Olmo2", "Granite"])
def test_the_last_branch_handed_to_the_next_layer(name):
    """`enable_residual_carry` over such layers: the norm behind the MLP runs with the next layer's first norm."""
    model = tiny(name, num_hidden_layers=3, **({"residual_multiplier": 0.22} if name == "Granite" else {})).to(DEV)
    ids = torch.arange(40, device=DEV)[None] % 160
    pos = torch.arange(40, device=DEV)[None]
    weights = torch.randn(1, 40, 160, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    want, wgrads = run(model, ids, pos, weights)
    fused.fuse_model(model)
    try:
        assert fused.enable_residual_carry(model) == 3
        timer = prl._capi.KernelTimer()
        prl._capi.set_timer(timer)
        got, grads = run(model, ids, pos, weights)
        prl._capi.set_timer(None)
        seen = timer.summary()
        # nothing of a layer's norms is left to the norm kernels but the first layer's own (if it has one)
        assert seen["prl_block_norms_fwd"]["launches"] == 6
        assert seen.get("prl_rmsnorm_fwd", {"launches": 0})["launches"] <= 1 + 2 * 3  # (query / key norms)
        assert fused.enable_residual_carry(model, False) == 0
        assert (T.forward(model, ids, pos) - want).abs().max() <= 2000 * 2.0**-24 * want.abs().max()
    finally:
        prl._capi.set_timer(None)
        fused.unfuse_model(model)
    assert not hasattr(model.model.layers[0], "_prl_carry")
    assert (got - want).abs().max() <= 2000 * 2.0**-24 * want.abs().max()
    for n, g in grads.items():
        assert (g - wgrads[n]).norm() <= 2000 * 2.0**-24 * wgrads[n].norm() + 1e-12, n


def test_two_families_in_one_process_keep_their_own_pairs():
    first, second = tiny("Qwen3").to(DEV), tiny("Glm4").to(DEV)
    ids, pos = torch.arange(32, device=DEV)[None], torch.arange(32, device=DEV)[None]
    want = [T.forward(m, ids, pos) for m in (first, second)]
    try:
        for m in (first, second):
            fused.fuse_model(m)
        for m, w in zip((second, first), reversed(want)):
            assert (T.forward(m, ids, pos) - w).abs().max() <= 2000 * 2.0**-24 * w.abs().max()
    finally:
        for m in (first, second):
            fused.unfuse_model(m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_step_of_a_model_with_norms_on_either_side(dtype):
    """Rotary embedding from positions, norms around the blocks, clipping: one `train_step`, fused against not."""
    base = tiny("Glm4", vocab_size=2048).to(DEV, dtype)
    gen = torch.Generator().manual_seed(5)
    t = 64
    mbs = [{
        "input_ids": torch.randint(0, 2048, (1, t), generator=gen),
        "position_ids": torch.cat([torch.arange(n) for n in (20, 12, 32)]).unsqueeze(0),
        "advantages": torch.randn(1, t, generator=gen),
        "logprobs": -7.6 + 0.3 * torch.randn(1, t, generator=gen),
        "loss_mask": torch.rand(1, t, generator=gen) < 0.7,
        "temperature": 0.9,
    } for _ in range(3)]
    results = []
    for fuse in (False, True):
        model = copy.deepcopy(base)
        if fuse:
            fused.fuse_model(model)
        timer = prl._capi.KernelTimer()
        prl._capi.set_timer(timer)
        try:
            opt = torch.optim.SGD(model.parameters(), lr=1.0)
            res = T.train_step(model, opt, copy.deepcopy(mbs), prl.LossConfig(), max_norm=1e-3, device=DEV)
        finally:
            prl._capi.set_timer(None)
            if fuse:
                fused.unfuse_model(model)
        results.append((res, {n: (p.detach().double() - q.detach().double()) for (n, p), (_, q) in
                              zip(model.named_parameters(), base.named_parameters())}, timer.summary()))
    (r0, d0, s0), (r1, d1, s1) = results
    for name in ("prl_rope_positions", "prl_block_norms_fwd", "prl_block_norms_bwd"):
        assert name in s1 and name not in s0
    assert "prl_grad_clip" in s0 and "prl_grad_clip" in s1
    # bf16: each of two layers rounds some ten intermediate tensors by up to 2^-8, which the fused form does not
    tol = 2000 * 2.0**-24 if dtype == torch.float32 else 20 * 2.0**-8
    assert abs(r1.grad_norm - r0.grad_norm) <= tol * r0.grad_norm and r0.grad_norm > 1e-3
    if dtype == torch.float32:  # the clipped step itself (in bf16 it drowns in the weights' own rounding)
        # weights of size up to 1 keep a step to 2^-24 of themselves on either side
        for n in d0:
            assert (d1[n] - d0[n]).norm() <= tol * d0[n].norm() + 2.0**-23 * d0[n].numel() ** 0.5, n
        total = torch.stack([d.norm() for d in d1.values()]).norm()
        assert abs(float(total) - 1e-3) <= 0.02 * 1e-3  # the update is as long as the clipping allows
