"""Optimizers and learning-rate schedules of the trainer
(counterparts of src/prime_rl/trainer/optim.py:9-57 and src/prime_rl/trainer/scheduler.py:7-105).

The schedules are written as one closed-form factor of the step instead of a
chain of torch schedulers; `tests/test_optim.py` checks that they trace the same
learning rates as the reference's composition of LinearLR / CosineAnnealingLR /
SequentialLR."""

from __future__ import annotations

import math
import operator
from typing import Any, Callable

import numpy as np
import torch
from torch import nn
from torch.optim.lr_scheduler import LambdaLR, LRScheduler


class FlatAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update over ONE flat fp32 parameter on the GPU (the master shard of
    `replica.FlatState`), as one HIP launch that also applies the clipping factor, writes the compute copy of the
    new weights and clears the gradient (`prl_adamw_flat`).  Learning-rate schedulers drive it like any optimizer."""

    def __init__(self, params: Any, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        if len(self.param_groups) != 1 or len(self.param_groups[0]["params"]) != 1:
            raise ValueError("FlatAdamW takes exactly one (flat) parameter")

    @torch.no_grad()
    def step_flat(self, grad: torch.Tensor, grad_scale: torch.Tensor | None = None,
                  compute_copy: torch.Tensor | None = None, zero_grad: bool = False) -> None:
        """One step with `grad` (fp32, same size as the parameter) times `grad_scale` (a 1-element device tensor,
        or None); `compute_copy` receives the new weights in its own dtype; `zero_grad` clears `grad`."""
        from . import _capi as C

        group = self.param_groups[0]
        p = group["params"][0]
        dev = C.require_device(p, grad, grad_scale, compute_copy)
        if p.dtype != torch.float32 or grad.dtype != torch.float32 or grad.numel() != p.numel() \
                or not (p.is_contiguous() and grad.is_contiguous()):
            raise ValueError("FlatAdamW: parameter and gradient must be contiguous fp32 tensors of one size")
        if compute_copy is not None and (compute_copy.numel() != p.numel() or not compute_copy.is_contiguous()):
            raise ValueError("FlatAdamW: the compute copy must be contiguous and as long as the parameter")
        state = self.state[p]
        if not state:
            state["step"] = 0
            state["exp_avg"] = torch.zeros_like(p)
            state["exp_avg_sq"] = torch.zeros_like(p)
        state["step"] += 1
        self._opt_called = True  # what torch's schedulers look at to tell a step has been taken
        b1, b2 = group["betas"]
        with C.on_device(dev), C.timed("prl_adamw_flat", dev):
            C.check(
                C.load().prl_adamw_flat(C.ptr(p), C.ptr(grad), C.ptr(state["exp_avg"]), C.ptr(state["exp_avg_sq"]),
                                        C.ptr(compute_copy), 0 if compute_copy is None else C.dtype_code(compute_copy),
                                        p.numel(), C.ptr(grad_scale), int(zero_grad), float(group["lr"]), float(b1),
                                        float(b2), float(group["eps"]), float(group["weight_decay"]), state["step"],
                                        C.stream_ptr(dev)),
                "prl_adamw_flat",
            )

    @torch.no_grad()
    def step(self, closure: Any = None) -> None:  # the plain Optimizer protocol: the parameter's own .grad
        p = self.param_groups[0]["params"][0]
        if p.grad is not None:
            self.step_flat(p.grad)


def setup_optimizer(config: Any, model: nn.Module, fused: bool | None = None, flat: bool = False) -> torch.optim.Optimizer:
    """The optimizer of src/prime_rl/trainer/optim.py:9-38 over `model.parameters()`.  `fused` asks torch for its
    one-kernel AdamW (same update rule) or for the per-operation one; left at None it is the one-kernel form
    wherever the parameters are on a GPU: over FSDP2's 311 sharded parameters of a 0.6B model the per-operation
    form costs the step 23 ms of small launches (135 -> 112 ms).  `flat=True` (one flat fp32 parameter on the
    GPU) gives `FlatAdamW`."""
    if config.type == "adamw" and flat:
        return FlatAdamW(model.parameters(), lr=config.lr, weight_decay=config.weight_decay,
                         betas=(config.betas1, config.betas2))
    if config.type == "sgd":
        return torch.optim.SGD(model.parameters(), lr=config.lr, weight_decay=config.weight_decay,
                               momentum=config.momentum, nesterov=config.nesterov)
    if config.type == "adamw":
        if fused is None:
            first = next(iter(model.parameters()), None)
            fused = bool(first is not None and first.is_cuda)
        return torch.optim.AdamW(model.parameters(), lr=config.lr, weight_decay=config.weight_decay,
                                 betas=(config.betas1, config.betas2), fused=fused)
    if config.type == "muon":
        raise NotImplementedError("the Muon optimizer comes from the `dion` package, which is not installed here")
    raise ValueError(f"Invalid optimizer type: {config.type}")


# --------------------------------------------------------------------------- gradient norm and clipping


_PIECE = np.dtype([("x", np.int64), ("n", np.int64), ("dtype", np.int32), ("reserved", np.int32)])  # prl_grad_piece


def _all_plain(grads: list[torch.Tensor]) -> bool:
    return set(map(type, grads)) <= {torch.Tensor}


def _sharding(grads: list[torch.Tensor]) -> list[Any] | None:
    """Process groups over which the squares of these gradients' local parts have to be added up: those of the mesh
    dimensions the gradients are sharded over ([] for plain tensors and for meshes of one rank).  None if they are
    not all plain, or all DTensors of one mesh with one placement, sharded or replicated, per mesh dimension."""
    if _all_plain(grads):
        return []
    spread = [g for g in grads if hasattr(g, "to_local")]
    if not spread:
        return []
    mesh, kinds = spread[0].device_mesh, [p.is_shard() for p in spread[0].placements]
    for g in grads:
        if not hasattr(g, "to_local") or g.device_mesh != mesh or [p.is_shard() for p in g.placements] != kinds \
                or any(p.is_partial() for p in g.placements):
            return None
    return [mesh.get_group(i) for i, shard in enumerate(kinds) if shard and mesh.size(i) > 1]


def _local_parts(grads: list[torch.Tensor]) -> list[torch.Tensor]:
    return grads if _all_plain(grads) else [g.to_local() if hasattr(g, "to_local") else g for g in grads]


def _one_device(parts: list[torch.Tensor]) -> torch.device:
    """The one HIP device of all of them (a RuntimeError says what is wrong otherwise)."""
    from . import _capi as C

    index = set(map(torch.Tensor.get_device, parts))
    return parts[0].device if len(index) == 1 and index != {-1} else C.require_device(*parts)


def _is_one_run(g: torch.Tensor) -> bool:
    """Whether a tensor's elements fill one run of memory, in whatever order of its dimensions."""
    if g.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((st, n) for st, n in zip(g.stride(), g.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _overlap(at: np.ndarray, size: np.ndarray) -> bool:
    """Whether any two runs of `size` bytes (none empty) at these addresses share memory."""
    order = np.argsort(at)
    return bool(((at + size)[order[:-1]] > at[order[1:]]).any())


def clip_grad_norm_supported(grads: list[torch.Tensor]) -> bool:
    """Whether `clip_grad_norm_` takes these gradients: bf16 or fp32, each one run of memory and no two the same, on one
    HIP device, plain or DTensors of one mesh that are sharded or replicated alike."""
    if not grads:
        return True
    if _sharding(grads) is None:
        return False
    parts = _local_parts(grads)
    index = set(map(torch.Tensor.get_device, parts))
    if len(index) != 1 or index == {-1} or not set(map(_DTYPE, parts)) <= _TYPES \
            or not all(g.layout is torch.strided and _is_one_run(g) for g in parts):
        return False
    runs = np.array([(g.data_ptr(), g.nbytes) for g in parts if g.numel()], dtype=np.int64).reshape(-1, 2)
    return not _overlap(runs[:, 0], runs[:, 1])


_GRAD, _DTYPE = operator.attrgetter("grad"), operator.attrgetter("dtype")
_TYPES = {torch.float32, torch.bfloat16}


def _pieces(grads: list[torch.Tensor], in_place: bool) -> np.ndarray:
    """The gradients as runs of memory: an array of `prl_grad_piece`.  Runs that touch end to end become one."""
    # (hundreds of tensors a call, so whole-list operations: 311 gradients take 76 us on the host, a loop took 106)
    types = list(map(_DTYPE, grads))
    kinds = set(types)
    try:
        at, whole = list(map(torch.Tensor.data_ptr, grads)), all(map(torch.Tensor.is_contiguous, grads))
    except RuntimeError:  # a layout without one address
        at, whole = [], False
    if not whole or not kinds <= _TYPES:
        for g in grads:
            if g.dtype not in _TYPES or g.layout is not torch.strided or not _is_one_run(g):
                raise ValueError("gradients must be dense float32 or bfloat16 tensors that fill one run of memory, got "
                                 f"{g.dtype} {g.layout} of shape {tuple(g.shape)}" +
                                 (f" with strides {g.stride()}" if g.layout is torch.strided else ""))
    table = np.zeros(len(grads), dtype=_PIECE)
    table["x"], table["n"] = at, list(map(torch.Tensor.numel, grads))
    if torch.bfloat16 in kinds:  # (PRL_F32 = 0, PRL_BF16 = 1)
        table["dtype"] = 1 if len(kinds) == 1 else [t is torch.bfloat16 for t in types]
    table = table[table["n"] > 0]
    if len(table) > 1:
        size = table["n"] * (4 - 2 * table["dtype"])
        at = table["x"]
        if in_place and _overlap(at, size):
            raise ValueError("clip_grad_norm_: two gradients share memory (a parameter given twice?)")
        first = np.flatnonzero(np.r_[True, ((at + size)[:-1] != at[1:]) | (table["dtype"][:-1] != table["dtype"][1:])])
        if len(first) < len(table):
            n = np.add.reduceat(table["n"], first)
            table = table[first]
            table["n"] = n
    return table


def _written(tensors: list[torch.Tensor]) -> None:
    """Counts a write to each of them, as torch's in-place operations do: a graph that has kept one notices."""
    count = torch.autograd.graph.increment_version
    try:
        count(tensors)
    except RuntimeError:  # (inference tensors count none; one counted twice is no harm)
        count([t for t in tensors if not t.is_inference()])


def _norm_kind(norm_type: float) -> int:
    from . import _capi as C

    if float(norm_type) == 2.0:
        return C.NORM_L2
    if float(norm_type) == math.inf:
        return C.NORM_MAX
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")


def _norm_and_factor(table: np.ndarray, dev: torch.device, kind: int, max_norm: float,
                     groups: list[Any]) -> torch.Tensor:
    """fp32 [2] on the device: the norm over `groups` and the clipping factor."""
    from . import _capi as C
    from .utils import _all_reduce

    lib = C.load()
    out = torch.empty(2, dtype=torch.float32, device=dev)
    at, n = table.ctypes.data, len(table)
    size = lib.prl_grad_norm_workspace_bytes(at, n)
    ws = torch.empty(size // 8 + 1, dtype=torch.float64, device=dev)  # the last one: the total
    total = ws.data_ptr() + size
    st = C.stream_ptr(dev)
    C.check(lib.prl_grad_norm(at, n, kind, max_norm, total, out.data_ptr(), out.data_ptr() + 4, ws.data_ptr(), size,
                              st), "prl_grad_norm")
    if groups:
        whole = ws[-1:]
        for group in groups:
            _all_reduce(whole, torch.distributed.ReduceOp.MAX if kind == C.NORM_MAX else torch.distributed.ReduceOp.SUM,
                        group)
        C.check(lib.prl_grad_norm_finish(total, 1, kind, max_norm, 0, out.data_ptr(), out.data_ptr() + 4, st),
                "prl_grad_norm_finish")
    return out


@torch.no_grad()
def grad_norm(grads: Any, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (2 or inf) of all these tensors (or of one) together, an fp32 scalar on their device, as
    torch.nn.utils.get_total_norm; squares are added in fp64 and nothing is copied to the host.  DTensors count with
    all ranks' shards."""
    from . import _capi as C

    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    kind = _norm_kind(norm_type)
    if not grads:
        return torch.tensor(0.0)
    groups = _sharding(grads)
    if groups is None:
        raise ValueError("grad_norm: plain tensors, or DTensors of one mesh placed alike (sharded or replicated)")
    parts = _local_parts(grads)
    dev = _one_device(parts)
    table = _pieces(parts, in_place=False)
    with C.on_device(dev), C.timed("prl_grad_norm", dev):
        return _norm_and_factor(table, dev, kind, 0.0, groups)[0]


@torch.no_grad()
def clip_grad_norm_(parameters: Any, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ (src/prime_rl/trainer/rl/train.py:336-338) on the package's kernels: every
    gradient is multiplied in place by min(1, max_norm / (norm + 1e-6)); returns the norm before, an fp32 scalar on the
    device.  One read of the gradients for the norm; the second pass leaves them untouched when there is nothing to
    clip.  No host synchronisation (`error_if_nonfinite` looks at the norm and has one).  FSDP2's sharded gradients
    are taken with one all-reduced scalar per sharded mesh dimension.  bf16 and fp32 gradients may be mixed;
    `norm_type` is 2 or inf; a gradient given twice, or sharing memory with another, is refused."""
    from . import _capi as C

    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [g for g in map(_GRAD, params) if g is not None]
    kind = _norm_kind(norm_type)
    if not grads:
        return torch.tensor(0.0)
    plain = _all_plain(grads)
    groups = [] if plain else _sharding(grads)
    if groups is None:
        raise ValueError("clip_grad_norm_: plain gradients, or DTensors of one mesh placed alike (sharded or replicated)")
    parts = grads if plain else _local_parts(grads)
    dev = _one_device(parts)
    table = _pieces(parts, in_place=True)
    lib, at, n = C.load(), table.ctypes.data, len(table)
    if not groups and not error_if_nonfinite:
        norm = torch.empty((), dtype=torch.float32, device=dev)
        size = lib.prl_grad_norm_workspace_bytes(at, n)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        C.run(lib.prl_grad_clip, "prl_grad_clip", dev, at, n, kind, float(max_norm), norm.data_ptr(), ws.data_ptr(), size,
              C.stream_ptr(dev))
        _written(grads)
        return norm
    with C.on_device(dev), C.timed("prl_grad_clip", dev):
        out = _norm_and_factor(table, dev, kind, float(max_norm), groups)
        if error_if_nonfinite and not math.isfinite(float(out[0])):
            raise RuntimeError(f"The total norm of order {norm_type} of the gradients is not finite, so they cannot be clipped")
        C.check(lib.prl_grad_scale(at, n, out.data_ptr() + 4, C.stream_ptr(dev)), "prl_grad_scale")
    _written(grads)
    if parts is not grads:
        _written(parts)
    return out[0]


def _floor_factor(lr: float, min_lr: float) -> float:
    return min_lr / lr if min_lr > 0 else 1e-8


def linear_factor(max_steps: int | None, warmup_steps: int, decay_steps: int, lr: float, min_lr: float) -> Callable[[int], float]:
    """Warm-up, plateau, linear decay (src/prime_rl/trainer/scheduler.py:12-47)."""
    assert warmup_steps > 0 or decay_steps > 0, "Either warmup steps or decay steps must be specified for a linear scheduler"
    floor = _floor_factor(lr, min_lr)
    decay_start = None
    if decay_steps > 0:
        assert max_steps is not None, "max_steps must be specified when specifying decay_steps"
        decay_start = max_steps - decay_steps
        assert decay_start >= warmup_steps

    def factor(step: int) -> float:
        if step < warmup_steps:
            return floor + (1.0 - floor) * step / warmup_steps
        if decay_start is None or step < decay_start:
            return 1.0
        span = decay_steps - 1  # the reference decays over decay_steps - 1 intervals
        k = min(step - decay_start, span)
        return 1.0 + (floor - 1.0) * (k / span if span > 0 else 1.0)

    return factor


def cosine_factor(max_steps: int | None, warmup_steps: int, lr: float, min_lr: float) -> Callable[[int], float]:
    """Warm-up, then half a cosine down to min_lr (src/prime_rl/trainer/scheduler.py:50-75)."""
    assert max_steps is not None, "max_steps must be specified when specifying decay_steps"
    floor = _floor_factor(lr, min_lr)
    t_max = max_steps - warmup_steps

    def factor(step: int) -> float:
        if step < warmup_steps:
            return floor + (1.0 - floor) * step / warmup_steps
        k = step - warmup_steps
        return (min_lr + (lr - min_lr) * (1.0 + math.cos(math.pi * k / t_max)) / 2.0) / lr

    return factor


def setup_scheduler(optimizer: torch.optim.Optimizer, config: Any, max_steps: int | None, lr: float) -> LRScheduler:
    if config.type == "constant":
        return LambdaLR(optimizer, lambda step: 1.0)
    if config.type == "linear":
        return LambdaLR(optimizer, linear_factor(max_steps, config.warmup_steps, config.decay_steps, lr, config.min_lr))
    if config.type == "cosine":
        return LambdaLR(optimizer, cosine_factor(max_steps, config.warmup_steps, lr, config.min_lr))
    raise ValueError(f"Invalid scheduler type: {config.type}")
