"""What the operators beside the fused block kernels refuse before a launch, and their host-side parts; no GPU."""

import ctypes
import math

import pytest
import torch

import prime_rl_cse_amd as prl  # noqa: F401
from prime_rl_cse_amd import _capi as C
from prime_rl_cse_amd import fused, optim

ONE, NULL = 16, None  # an address that is never followed: validation fails first


def test_host_tensors_are_refused():
    q, pos = torch.zeros(1, 2, 3, 8), torch.arange(3)
    with pytest.raises(RuntimeError):
        fused.rope_at_positions(q, q, pos, torch.ones(4))
    with pytest.raises(RuntimeError):
        fused.block_norms(q, q, torch.ones(8), torch.ones(8))
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_([p], 1.0)
    assert not fused.rope_at_positions_supported(q, q, pos, torch.ones(4))
    assert not fused.block_norms_supported(q, q) and not optim.clip_grad_norm_supported([p.grad])


def test_rope_positions_entry_refuses():
    lib = C.load()
    s = (C.c_int64 * 6)(24, 24, 8, 24, 24, 8)

    def call(q=ONE, qo=ONE, qs=s, hq=1, k=NULL, ko=NULL, ks=None, hk=0, pos=ONE, freq=ONE, r=8, dtype=0, b=1, t=3, d=8):
        return lib.prl_rope_positions(q, qo, qs, hq, k, ko, ks, hk, pos, 1, 0, 1, freq, 0, r, 0, 1.0, dtype, b, t, d, 0, None)

    assert call(t=0) == 0 and call(b=0) == 0 and call(hq=0) == 0
    for bad in (dict(r=7), dict(r=0), dict(r=10), dict(dtype=2), dict(t=-1), dict(hq=-1), dict(pos=NULL), dict(freq=NULL),
                dict(q=NULL), dict(qo=NULL), dict(hk=1), dict(q=18), dict(b=1 << 16, t=1 << 15), dict(b=1 << 40, t=1 << 40),
                dict(hq=1 << 20)):
        assert call(**bad) == -1, bad
        assert lib.prl_last_error()
    assert lib.prl_rope_positions_supported(1, 128, 64) == 1 and lib.prl_rope_positions_supported(1, 16384, 8194) == 0


def test_block_norms_entries_refuse():
    lib = C.load()

    def fwd(x=ONE, b=ONE, w1=ONE, w2=ONE, kind=0, gate=NULL, hid=ONE, hs=16, y=ONE, ys=16, dtype=0, rows=2, h=16):
        return lib.prl_block_norms_fwd(x, 16, b, 16, w1, w2, kind, gate, 0, 1.0, 0.0, 1e-6, 1e-6, hid, hs, y, ys, NULL, NULL,
                                       dtype, rows, h, None)

    assert fwd(rows=0) == 0
    for bad in (dict(x=NULL), dict(b=NULL), dict(hid=NULL), dict(y=NULL), dict(kind=1), dict(kind=4), dict(hs=8), dict(ys=15),
                dict(dtype=5), dict(h=0), dict(h=8193), dict(rows=-1), dict(x=18)):
        assert fwd(**bad) == -1, bad

    def bwd(w1=ONE, w2=ONE, kind=0, gate=NULL, r1=ONE, r2=ONE, gy=ONE, gx=ONE, gw1=ONE, gw2=ONE, gg=NULL, ggs=16, ws=ONE,
            size=1 << 20, gxs=16):
        return lib.prl_block_norms_bwd(ONE, 16, ONE, 16, w1, w2, kind, gate, 16, 1.0, 0.0, r1, r2, NULL, 0, gy, 16, gx, gxs,
                                       ONE, 16, gw1, gw2, gg, ggs, 0, 2, 16, ws, size, None)

    for bad in (dict(r1=NULL), dict(r2=NULL), dict(gy=NULL), dict(gx=NULL), dict(w1=NULL), dict(w2=NULL), dict(gg=ONE),
                dict(ws=NULL), dict(size=64), dict(ws=20), dict(gxs=8), dict(kind=3, gate=ONE, gg=ONE, ggs=8),
                dict(kind=2, gate=ONE, gg=ONE, ggs=0)):
        assert bwd(**bad) == -1, bad
    assert lib.prl_block_norms_bwd_workspace_bytes(1, 100, 9000) == 0
    assert lib.prl_block_norms_bwd_workspace_bytes(1, 0, 64) > 0


def test_grad_entries_refuse():
    lib = C.load()
    ok = (C.GradPiece * 2)((16, 10, 0, 0), (128, 0, 1, 0))
    assert lib.prl_grad_norm_workspace_bytes(ok, 2) == 8 and lib.prl_grad_norm_workspace_bytes(ok, 0) == 8
    for bad in ((16, -1, 0, 0), (16, 4, 2, 0), (0, 4, 0, 0), (18, 4, 0, 0), (17, 4, 1, 0), (16, 1 << 43, 1, 0)):
        t = (C.GradPiece * 1)(bad)
        assert lib.prl_grad_norm(t, 1, 0, 1.0, ONE, ONE, ONE, ONE, 1 << 20, None) == -1
        assert lib.prl_grad_scale(t, 1, ONE, None) == -1
        assert lib.prl_grad_clip(t, 1, 0, 1.0, ONE, ONE, 1 << 20, None) == -1
        assert lib.prl_grad_norm_workspace_bytes(t, 1) == 0
    assert lib.prl_grad_norm(ok, 2, 2, 1.0, ONE, ONE, ONE, ONE, 64, None) == -1
    assert lib.prl_grad_norm(ok, 2, 0, 1.0, None, None, None, ONE, 64, None) == -1
    assert lib.prl_grad_norm(ok, 2, 0, 1.0, ONE, ONE, ONE, ONE, 4, None) == -1
    assert lib.prl_grad_norm(ok, -1, 0, 1.0, ONE, ONE, ONE, ONE, 64, None) == -1
    assert lib.prl_grad_clip(ok, 2, 0, 1.0, None, ONE, 64, None) == -1 and lib.prl_grad_clip(ok, 2, 0, 1.0, ONE, ONE, 4, None) == -1
    assert lib.prl_grad_scale(ok, 2, None, None) == -1 and lib.prl_grad_scale(ok, 0, ONE, None) == 0
    assert lib.prl_grad_norm_finish(None, 1, 0, 1.0, ONE, ONE, ONE, None) == -1
    big = (C.GradPiece * 300)(*[(16, 1 << 20, i % 2, 0) for i in range(300)])
    assert lib.prl_grad_norm_workspace_bytes(big, 300) > 8


def test_gradients_as_runs_of_memory():
    a = torch.randn(6, 4)
    table = optim._pieces([a[:2], a[2:], a.new_zeros(0), torch.randn(3).bfloat16()], True)
    assert [(int(p["n"]), int(p["dtype"])) for p in table] == [(24, C.PRL_F32), (3, C.PRL_BF16)]
    assert table.dtype.itemsize == ctypes.sizeof(C.GradPiece) and len(optim._pieces([a.new_zeros(0)], True)) == 0
    assert len(optim._pieces([a[3:], a[:3]], True)) == 2  # touching, but not in order
    assert optim._is_one_run(a.t()) and optim._is_one_run(torch.randn(3, 4, 5).permute(2, 0, 1))
    assert not optim._is_one_run(a[:, :3]) and not optim._is_one_run(a.expand(2, 6, 4))
    for bad in ([a, a], [a, a[1:2]], [a[:, 1]], [a.half()], [a.to_sparse()]):
        with pytest.raises(ValueError):
            optim._pieces(bad, True)
    optim._pieces([a, a[1:2]], False)  # reading twice is no harm


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default"}, {"rope_type": "linear", "factor": 3.0},
    {"rope_type": "dynamic", "factor": 2.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 1024, "beta_fast": 16.0, "beta_slow": 2.0,
     "attention_factor": 1.25},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 1024, "mscale": 1.0, "mscale_all_dim": 0.7},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 1024},
    {"rope_type": "longrope", "short_factor": [1.0 + 0.1 * i for i in range(32)],
     "long_factor": [1.0 + i for i in range(32)], "original_max_position_embeddings": 1024},
])
@pytest.mark.parametrize("seq_len", [None, 1000, 9000])
def test_frequencies_are_those_a_model_of_the_same_config_uses(scaling, seq_len):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    kind = scaling["rope_type"]
    config = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=64, max_position_embeddings=4096,
                         rope_parameters={"rope_theta": 5e5, **scaling})
    got, amplitude = fused.rope_frequencies(64, 5e5, scaling, 4096, seq_len)
    if kind == "default":
        want, attention = 5e5 ** (-torch.arange(32, dtype=torch.float64) / 32), 1.0
    else:
        want, attention = ROPE_INIT_FUNCTIONS[kind](config, torch.device("cpu"), seq_len=seq_len)
    # fp32 powers there (a few roundings of the exponent, times ln 5e5 = 13), one rounding here
    assert torch.allclose(got.double(), want.double(), rtol=4e-6, atol=0)
    assert math.isclose(amplitude, attention, rel_tol=1e-6)


def test_frequencies_refuse():
    for args in ((7,), (0,), (8, 1e4, {"rope_type": "linear"}), (8, 1e4, {"rope_type": "yarn", "factor": 2.0}),
                 (8, 1e4, {"rope_type": "nonsense"}), (8, 1e4, {"rope_type": "llama3", "factor": 2.0}, 64),
                 (8, 1e4, {"rope_type": "longrope", "short_factor": [1.0], "long_factor": [1.0]}, 64)):
        with pytest.raises(ValueError):
            fused.rope_frequencies(*args)
