"""What `fuse_model` reads off a model family before it rebinds anything: the pairs of its rotary embedding, the steps
of its decoder layer, the form of its norms.  Host only; the kernels' side is tests/test_gpu_families.py."""

import sys

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import fused


def tiny(name, **kw):
    import transformers
    from transformers import AutoModelForCausalLM

    args = dict(hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                head_dim=16, vocab_size=160, pad_token_id=0, bos_token_id=1, eos_token_id=2, max_position_embeddings=256,
                attn_implementation="eager", use_cache=False)
    args.update(kw)
    torch.manual_seed(0)
    return AutoModelForCausalLM.from_config(getattr(transformers, name + "Config")(**args))


KINDS = {"Qwen3": ("half", False), "Llama": ("half", False), "Glm4": ("interleaved", True), "Cohere": ("interleaved", True),
         "Helium": ("interleaved", True), "Glm4Moe": ("half", True), "Gemma2": ("half", False)}


@pytest.mark.parametrize("name", list(KINDS))
def test_pairs_of_the_rotary_embedding(name):
    model = tiny(name)
    kind, tagged = fused._rope_kind(sys.modules[type(model).__module__], model)
    assert (kind, bool(tagged)) == KINDS[name]


def test_a_family_that_does_something_else_is_left_alone():
    class Home:
        @staticmethod
        def rotate_half(x):
            return -x

        @staticmethod
        def apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim=1):
            return q * 2, k * 2

    assert fused._rope_kind(Home, tiny("Qwen3")) is None
    assert fused._rope_kind(Home, torch.nn.Linear(2, 2)) is None


STEPS = {
    "Glm4": ("input_layernorm", "post_self_attn_layernorm", None, "post_attention_layernorm", "post_mlp_layernorm", None),
    "Gemma2": ("input_layernorm", "post_attention_layernorm", None, "pre_feedforward_layernorm",
               "post_feedforward_layernorm", None),
    "Olmo2": (None, "post_attention_layernorm", None, None, "post_feedforward_layernorm", None),
    "Granite": ("input_layernorm", None, "residual_multiplier", "post_attention_layernorm", None, "residual_multiplier"),
}


@pytest.mark.parametrize("name", list(STEPS))
def test_steps_of_a_layer_with_norms_behind_its_blocks(name):
    layer = tiny(name).model.layers[0]
    assert not fused._is_plain_decoder_layer(layer)  # taken for one, the norms behind the blocks would be left out
    st = fused._layer_steps(layer)
    assert (st.pre1, st.post1, st.scale1, st.pre2, st.post2, st.scale2) == STEPS[name]


@pytest.mark.parametrize("name", ["Qwen3", "Qwen2", "Llama", "Glm"])
def test_plain_layers_stay_plain(name):
    layer = tiny(name).model.layers[0]
    assert fused._is_plain_decoder_layer(layer) and fused._layer_steps(layer) is None


def test_other_layers_are_left_alone():
    assert fused._layer_steps(tiny("Cohere").model.layers[0]) is None  # attention and MLP side by side
    assert fused._layer_steps(torch.nn.Linear(2, 2)) is None


def test_form_of_the_norms():
    assert fused._norm_form(tiny("Glm4").model.norm) == 0.0
    assert fused._norm_form(tiny("Gemma2").model.norm) == 1.0
    assert fused._norm_form(torch.nn.LayerNorm(8)) is None
    assert fused._norm_form(tiny("Cohere").model.norm) is None


@pytest.mark.parametrize("change", [None, "cos", "sin", "positions", "other"])
def test_tables_that_were_changed_are_not_replaced_by_positions(change, monkeypatch):
    """The positions left on a rotary module's cos stand for its tables only as long as these are what it returned."""
    taken = []
    monkeypatch.setattr(fused, "rope_at_positions_supported", lambda *a: True)
    monkeypatch.setattr(fused, "rope_at_positions", lambda q, k, *a, **kw: taken.append("positions") or (q, k))
    rotate = fused._family_rope(lambda q, k, cos, sin: taken.append("tables") or (q, k), "interleaved")
    rotary = tiny("Glm4").model.rotary_emb
    rotary._prl_torch_forward = rotary.forward
    q, k, pos = torch.randn(1, 2, 5, 16), torch.randn(1, 1, 5, 16), torch.arange(5)[None]
    cos, sin = fused._tagged_rotary_forward(rotary, q, pos)
    if change == "other":
        sin = sin.clone()
    elif change:
        {"cos": cos, "sin": sin, "positions": pos}[change].mul_(2)
    rotate(q, k, cos, sin)
    assert taken == ["tables" if change else "positions"]
    taken.clear()
    with torch.inference_mode():  # (tensors that count no writes)
        rotate(q, k, *fused._tagged_rotary_forward(rotary, q, pos))
    assert taken == ["tables"]


def test_form_of_a_norm_is_asked_of_the_module_itself():
    """A class may leave its weight out of some of its instances."""
    class Norm(torch.nn.Module):
        def __init__(self, scaled):
            super().__init__()
            self.eps = 1e-6
            self.weight = torch.nn.Parameter(torch.ones(8)) if scaled else None

        def forward(self, x):
            y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.eps)
            return y if self.weight is None else y * self.weight

    assert fused._norm_form(Norm(True)) == 0.0
    assert fused._norm_form(Norm(False)) is None
    assert fused._norm_form(Norm(True)) == 0.0
