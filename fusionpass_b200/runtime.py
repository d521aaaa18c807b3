"""Plan executor: ``execute_plan`` with the reference signature and semantics.

Reference: ``python/fusionpass/runtime.py:21-60``.  Unfused ``torch`` steps run
as eager PyTorch ops; fused steps (``kind: "triton"``, kept for plan
compatibility) go to ``kernels.launch_step``, i.e. to libfpkern.so on the
current CUDA stream.
"""

from __future__ import annotations

import torch

from . import block
from .kernels import check_device as _check_device
from .kernels import launch_step, load_kernels
from .validate import validate_plan

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "i32": torch.int32}

__all__ = ["execute_plan", "load_kernels", "validate_plan", "_run_torch", "_run_fused", "_check_device",
           "_DTYPES"]


def _run_torch(step: dict, ops: list) -> torch.Tensor:
    op, attrs = step["op"], step["attrs"]
    if op == "add":
        return torch.add(ops[0], ops[1])
    if op == "mul":
        return torch.mul(ops[0], ops[1])
    if op == "scale":
        return ops[0] * attrs["factor"]
    if op == "relu":
        return torch.relu(ops[0])
    if op == "exp":
        return torch.exp(ops[0])
    if op == "softmax":
        return torch.softmax(ops[0], dim=attrs["axis"])
    if op == "matmul":
        return torch.matmul(ops[0], ops[1])
    if op == "transpose":
        return ops[0].transpose(-1, -2)
    # extension steps (planner extensions=True)
    if op == "gelu":
        return torch.nn.functional.gelu(ops[0])
    if op == "linear":
        return torch.nn.functional.linear(ops[0], ops[1], ops[2] if len(ops) == 3 else None)
    if op == "layer_norm":
        w, b = (ops[1], ops[2]) if len(ops) == 3 else (None, None)
        if ops[0].is_cuda and len(attrs["normalized_shape"]) == 1:
            # over the last axis: the libfpkern kernel (None if it does not take the shape)
            from . import fpkern
            y = fpkern.layer_norm(ops[0], w, b, attrs["eps"])
            if y is not None:
                return y
        return torch.nn.functional.layer_norm(ops[0], attrs["normalized_shape"], w, b, attrs["eps"])
    if op == "add_layer_norm":
        # layer_norm of the sum of the first n_addends operands (the add chain that fed it)
        k = attrs["n_addends"]
        w, b = (ops[k], ops[k + 1]) if len(ops) == k + 2 else (None, None)
        if ops[0].is_cuda:
            from . import fpkern
            y = fpkern.add_layer_norm(ops[:k], w, b, attrs["eps"], shape=step.get("shape"))
            if y is not None:
                return y
        x = ops[0]
        for t in ops[1:k]:
            x = x + t
        return torch.nn.functional.layer_norm(x, attrs["normalized_shape"], w, b, attrs["eps"])
    if op == "rms_norm":
        return _rms_norm(ops[:1], ops[1] if len(ops) == 2 else None, attrs["eps"], step.get("shape"), False)[0]
    if op == "linear_q8":
        x, w, ws = ops[:3]
        b = ops[3] if len(ops) == 4 else None
        if not x.is_cuda:
            return block.linear_q8(x, w, ws, b)
        from . import fpkern
        q, scale = fpkern.quantize_q8(x)
        return fpkern.linear_q8(q, scale, w, ws, b, out_dtype=x.dtype)
    if op == "score_attention":
        return _score_attention(step, ops)
    if op == "reshape":
        return ops[0].reshape(attrs["shape"])
    if op == "cat":
        return torch.cat(ops, dim=attrs["dim"])
    if op == "narrow":
        return ops[0].narrow(attrs["dim"], attrs["start"], attrs["length"])
    if op == "permute":
        return ops[0].permute(*attrs["dims"])
    raise ValueError(f"unknown torch op in plan: {op}")


def _rms_norm(addends: list, weight, eps: float, shape, keep: bool) -> tuple:
    """(norm of the addends' sum, the sum if ``keep``)."""
    if addends[0].is_cuda:
        from . import fpkern
        r = fpkern.add_rms_norm(addends, weight, eps, shape=shape, return_sum=keep)
        return r if keep else (r, None)
    total = addends[0].float()
    for t in addends[1:]:
        total = total + t.float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight.float()
    return y.to(addends[0].dtype), total.to(addends[0].dtype)


def _run_norm(step: dict, ops: list) -> tuple:
    """``add_rms_norm`` / ``rms_norm_linear_q8``: (result, the sum where the step keeps it)."""
    attrs = step["attrs"]
    n, keep = attrs["n_addends"], "extra_result" in step
    addends, rest = ops[:n], ops[n:]
    weight = rest.pop(0) if attrs["affine"] else None
    if step["op"] == "add_rms_norm":
        return _rms_norm(addends, weight, attrs["eps"], step.get("shape"), keep)
    w, ws = rest[:2]
    b = rest[2] if len(rest) == 3 else None
    shape = list(step["shape"][:-1]) + [w.shape[1]] if "shape" in step else None
    if addends[0].is_cuda:
        from . import fpkern
        q, scale, *kept = fpkern.rms_norm_q8(addends, weight, attrs["eps"], shape=shape, return_sum=keep)
        y = fpkern.linear_q8(q, scale, w, ws, b, out_dtype=addends[0].dtype)
        return y, kept[0] if keep else None
    y, total = _rms_norm(addends, weight, attrs["eps"], shape, keep)
    return block.linear_q8(y, w, ws, b), total


def _score_attention(step: dict, ops: list) -> torch.Tensor:
    attrs = step["attrs"]
    kw = {k: attrs[k] for k in ("softcap", "causal", "window", "prefix") if k in attrs}
    kw.update(zip(attrs.get("optional", ()), ops[3:]))
    if not ops[0].is_cuda:
        return block.score_attention(*ops[:3], attrs["scale"], **kw)
    from . import fpkern
    layout = attrs.get("out_layout")
    if layout is not None:
        # stored with heads and sequence swapped, as the heads merge that follows reads it
        perm = [int(i) for i in layout]
        if perm != [0, 2, 1, 3]:
            raise ValueError(f"out_layout {layout} of a score_attention step is not [0, 2, 1, 3]")
        q = ops[0]
        kw["out"] = torch.empty([q.shape[i] for i in perm], dtype=q.dtype, device=q.device).permute(*perm)
    return fpkern.score_attention(*ops[:3], attrs["scale"], **kw)


def _run_fused(step: dict, ops: list, kernels) -> torch.Tensor:
    return launch_step(step, ops, kernels)


_run_triton = _run_fused  # the reference's name for the same hook


def execute_plan(plan: dict, args: list, kernels=None, *, validate: bool = True):
    """Run ``plan`` on ``args``; returns the single output (or a tuple)."""
    if validate:
        validate_plan(plan)
    if plan.get("version") != 1:
        raise ValueError(f"unsupported plan version {plan.get('version')}")
    if len(args) != len(plan["inputs"]):
        raise ValueError(f"expected {len(plan['inputs'])} inputs, got {len(args)}")
    env = {}
    for spec, t in zip(plan["inputs"], args):
        # static shapes: the plan and its descriptors are specialised to them
        if list(t.shape) != spec["shape"] or t.dtype != _DTYPES[spec["dtype"]]:
            raise ValueError(f"{spec['name']}: expected {spec['dtype']}{spec['shape']}, "
                             f"got {t.dtype}{list(t.shape)}")
        env[spec["name"]] = t
    for step in plan["steps"]:
        ops = [env[o] for o in step["operands"]]
        kind = step["kind"]
        if kind == "torch" and step["op"] in ("add_rms_norm", "rms_norm_linear_q8"):
            env[step["result"]], kept = _run_norm(step, ops)
            if "extra_result" in step:
                env[step["extra_result"]] = kept
        elif kind == "torch":
            env[step["result"]] = _run_torch(step, ops)
        elif kind == "triton":
            env[step["result"]] = _run_fused(step, ops, kernels)
        else:
            raise ValueError(f"unknown step kind {kind}")
    outs = [env[o] for o in plan["outputs"]]
    return outs[0] if len(outs) == 1 else tuple(outs)
