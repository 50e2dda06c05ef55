"""What a training step of the MLP block needs around `ops.fused_swiglu_mlp` and its backward pass: norms with
gradients, the clipped gradient norm, AdamW over many tensors at once.

    layer_norm, rms_norm     autograd functions over the rows of any leading dimensions (bf16 or fp32)
    norm_swiglu_block        x + MLP(norm(x)) with autograd: the fused kernels forward and backward
    clip_grad_norm           [norm, factor] on the device, for `FusedAdamW` or `adamw_step`
    FusedAdamW               torch.optim.Optimizer over `adamw_step`, moments in 32 bits or 8

The reference is forward only (csrc/torch_bindings.cpp:38-50).  The raw operators are functions of the torch extension
`fused_mlp_module` (and `torch.ops.ASMLLM`); the arithmetic is in libfswiglu.so, without a CPU path.

`layer_norm` and `rms_norm` can be traced (fake tensors, torch.compile); the block, the clipped norm and the optimiser run as they
are, outside of traced graphs.  vmap, forward-mode and second derivatives are refused.

Capturing a backward pass into a CUDA graph: as with every autograd function, no graph of an earlier eager pass over the
same leaves may be alive then (drop its outputs first, and let the warm-up pass run on the capturing stream).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _lib():
    import fused_mlp_module

    return fused_mlp_module


def _norms(x: torch.Tensor):
    """The module's functions; where x is traced or has shapes alone, the dispatcher's ops, which have forms for that."""
    lib = _lib()  # registers the ops
    plain = type(x) in (torch.Tensor, torch.nn.Parameter) and x.device.type != "meta"
    return lib if plain and not torch.compiler.is_compiling() and not torch._C._len_torch_dispatch_stack() else torch.ops.ASMLLM


def _rows(x: torch.Tensor, d: int) -> torch.Tensor:
    x2 = x.reshape(-1, d)
    plain = (x2.stride(1) == 1 or d == 1) and (x2.stride(0) >= d or x2.size(0) <= 1)  # not rows that share memory
    return x2 if plain else x2.contiguous()


def _operand(x: torch.Tensor, d: int) -> torch.Tensor:
    """Rows as the MLP's kernels read them: contiguous, from a 16-byte boundary on."""
    x2 = x.reshape(-1, d).contiguous()
    return x2 if x2.data_ptr() % 16 == 0 else x2.clone()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows(x, x.size(-1))
        y, mean, rstd = _norms(x2).layer_norm_forward(x2, weight, bias, eps)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x2, weight, mean, rstd = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        # vectors' gradients have the weight's type; a bias alone says by itself
        fp32 = weight is None and ctx.bias_dtype == torch.float32
        dx, dw, db = _norms(x2).layer_norm_backward(_rows(dout, x2.size(1)), x2, mean, rstd, weight, need_b,
                                                    fp32_grads=fp32, weight_grad=need_w)
        return dx.view(dout.shape), dw, None if db is None else db.to(ctx.bias_dtype), None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        x2 = _rows(x, x.size(-1))
        y, rstd = _norms(x2).rms_norm_forward(x2, weight, eps)
        ctx.save_for_backward(x2, weight, rstd)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x2, weight, rstd = ctx.saved_tensors
        dx, dw = _norms(x2).rms_norm_backward(_rows(dout, x2.size(1)), x2, rstd, weight,
                                              weight_grad=ctx.needs_input_grad[1])
        return dx.view(dout.shape), dw, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) * rsqrt(var + eps) * weight + bias over the last dimension, with gradients."""
    return _LayerNorm.apply(x, weight, bias, eps)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * weight over the last dimension, with gradients."""
    return _RMSNorm.apply(x, weight, eps)


class _NormSwiGLUBlock(torch.autograd.Function):
    """Keeps x, norm(x) and the row statistics; gate and up projections are computed again in the backward pass."""

    @staticmethod
    def forward(ctx, x, norm_weight, norm_bias, W_gate, W_up, W_down, eps, layer):
        x2 = _operand(x, x.size(-1))
        mean = None
        if layer:
            n, mean, rstd = _lib().layer_norm_forward(x2, norm_weight, norm_bias, eps)
        else:
            n, rstd = _lib().rms_norm_forward(x2, norm_weight, eps)
        ctx.save_for_backward(x2, n, mean, rstd, norm_weight, W_gate, W_up, W_down)
        ctx.layer = layer
        return ops.fused_swiglu_mlp_bf16(n, W_gate, W_up, W_down, residual=x2).view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x2, n, mean, rstd, norm_weight, W_gate, W_up, W_down = ctx.saved_tensors
        d2 = _operand(dout, x2.size(1))
        dn, dwg, dwu, dwd = ops.swiglu_mlp_backward(n, W_gate, W_up, W_down, d2)
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        # the residual's gradient joins where dx is written
        if ctx.layer:
            dx, dw, db = _lib().layer_norm_backward(dn, x2, mean, rstd, norm_weight, need_b, d2, weight_grad=need_w)
        else:
            dx, dw = _lib().rms_norm_backward(dn, x2, rstd, norm_weight, d2, weight_grad=need_w)
            db = None
        return dx.view(dout.shape), dw, db, dwg, dwu, dwd, None, None


def norm_swiglu_block(x: torch.Tensor, norm_weight: torch.Tensor, norm_bias: torch.Tensor | None, W_gate: torch.Tensor,
                      W_up: torch.Tensor, W_down: torch.Tensor, eps: float = 1e-6, norm: str = "rms") -> torch.Tensor:
    """x + MLP(norm(x)) with gradients for x, the norm's vectors and the three matrices; all bf16.

    norm is "rms" (norm_bias None) or "layer".
    """
    if norm not in ("rms", "layer"):
        raise ValueError('norm must be "rms" or "layer"')
    if norm == "rms" and norm_bias is not None:
        raise ValueError("RMS norm has no bias")
    for name, t in (("norm_weight", norm_weight), ("norm_bias", norm_bias)):
        if t is not None and t.dtype != torch.bfloat16:
            raise RuntimeError(f"{name} must be a bfloat16 tensor, got {t.dtype}")
    args = (x, norm_weight, norm_bias, W_gate, W_up, W_down, eps, norm == "layer")
    if torch.compiler.is_compiling():
        return _block_as_it_is(*args)
    return _NormSwiGLUBlock.apply(*args)


@torch.compiler.disable
def _block_as_it_is(*args) -> torch.Tensor:
    """Where torch.compile leaves its graph."""
    return _NormSwiGLUBlock.apply(*args)


def clip_grad_norm(grads, max_norm: float) -> torch.Tensor:
    """[norm, factor] of the gradients of a list, on their device: factor = min(1, max_norm / (norm + 1e-6)), NaN where
    the norm is not finite.  Nothing is scaled here: the factor is adamw_step's grad_scale, which multiplies as it reads."""
    return _lib().grad_norm_clip([g if g.is_contiguous() else g.contiguous() for g in grads], max_norm)


def moments_to_float(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values of 8-bit moments: float8 codes times the scale of their block of 256."""
    return codes.reshape(-1).float().mul_(scales.repeat_interleave(256)[:codes.numel()]).view(codes.shape)


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) in one launch for all tensors of a kind.

    state_bits    32: fp32 moments.  8: float8 moments in blocks of 256 with a power-of-two scale, rounded stochastically
                  from `seed` (the same seed and steps give the same bits).
    master        keep an fp32 copy of bf16 parameters, from which the step computes.  Without it a bf16 parameter loses
                  what each step's rounding drops.
    max_grad_norm clip the 2-norm over all gradients; no host sync.  A step whose norm is not finite changes no tensor
                  (the step counts go on).  `last_grad_norm` holds [norm, factor] of the last step, on the device.
    capturable    keep learning rate and step count on the device (`group["lr_tensor"]`, `group["step_tensor"]`), so that a
                  captured `step()` can be replayed; then all parameters of a group take every step together.  Take one
                  step before the capture, which is refused without this.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, master: bool = True, max_grad_norm: float | None = None, seed: int = 0,
                 capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas must lie in [0, 1)")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError("max_grad_norm must not be negative")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.state_bits, self.master, self.max_grad_norm = state_bits, master, max_grad_norm
        self.seed, self.capturable = seed, capturable
        self.last_grad_norm = None

    def __getstate__(self) -> dict:
        """As the base class's, which would leave a copy or a pickled optimiser without what is set above."""
        mine = ("state_bits", "master", "max_grad_norm", "seed", "capturable", "last_grad_norm")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in mine}}

    def _init_state(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        master = self.master and p.dtype == torch.bfloat16
        if not state or (master and "master" not in state):
            self._refuse_capture(p.device)
        if not state:
            state["step"] = 0
            if self.state_bits == 8:
                scales = dict(dtype=torch.float32, device=p.device)
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float8_e5m2, device=p.device)
                state["exp_avg_scale"] = torch.zeros((p.numel() + 255) // 256, **scales)
                state["exp_avg_sq_scale"] = torch.zeros((p.numel() + 255) // 256, **scales)
            else:
                state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if master and "master" not in state:
            state["master"] = p.detach().float()
        return state

    @staticmethod
    def _refuse_capture(device: torch.device) -> None:
        if _capturing(device):
            raise RuntimeError("take one step before the capture: a captured one would start from zero each time")

    @torch.compiler.disable  # lists, dictionaries and kernels that write through pointers: torch.compile leaves its graph here
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, every = [], []
        for index, group in enumerate(self.param_groups):
            kinds: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("FusedAdamW does not take sparse gradients")
                g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                every.append(g)
                kinds.setdefault((p.device, p.dtype, g.dtype, self.state.get(p, {}).get("step", 0)), []).append((p, g))
            if self.capturable and kinds:
                # one count for the group: those with gradients are those with state, but for the first step's
                known = {p for p in group["params"] if self.state.get(p)}
                if len({(k[0], k[3]) for k in kinds}) > 1 or (known and known != {p for of in kinds.values() for p, _ in of}):
                    raise RuntimeError("with capturable=True all parameters of a group take every step together")
            work += [(index, group, key, tensors) for key, tensors in kinds.items()]
        if not work:
            return loss
        if not self.capturable and _capturing(work[0][2][0]):
            raise RuntimeError("a captured step needs capturable=True: replays would repeat this one's count and rounding")
        if len({key[0] for _, _, key, _ in work}) > 1 and self.max_grad_norm is not None:
            raise RuntimeError("max_grad_norm needs all gradients on one device")
        scale = None
        if self.max_grad_norm is not None:
            self.last_grad_norm = _lib().grad_norm_clip(every, self.max_grad_norm)
            scale = self.last_grad_norm[1:]
        stepped = set()
        for order, (index, group, (device, _, _, taken), tensors) in enumerate(work):
            states = [self._init_state(p) for p, _ in tensors]
            lr_tensor = step_tensor = None
            if self.capturable:
                if "step_tensor" not in group:
                    self._refuse_capture(device)
                    group["lr_tensor"] = torch.full((1,), float(group["lr"]), dtype=torch.float32, device=device)
                    group["step_tensor"] = torch.full((1,), taken, dtype=torch.int64, device=device)
                lr_tensor, step_tensor = group["lr_tensor"], group["step_tensor"]
                if not _capturing(device):
                    lr_tensor.fill_(float(group["lr"]))
                if index not in stepped:
                    step_tensor.add_(1)
                    stepped.add(index)
            eight = self.state_bits == 8
            _lib().adamw_step([p for p, _ in tensors], [g for _, g in tensors], [s["exp_avg"] for s in states],
                              [s["exp_avg_sq"] for s in states], taken + 1, group["lr"], *group["betas"], group["eps"],
                              group["weight_decay"], [s["master"] for s in states if "master" in s],
                              [s["exp_avg_scale"] for s in states] if eight else [],
                              [s["exp_avg_sq_scale"] for s in states] if eight else [], scale,
                              # each launch of a step rounds by bits of its own
                              self.seed ^ (order * 0x61C88647 % 0x7FFFFFFF << 32), lr_tensor, step_tensor)
            if not self.capturable:
                for s in states:
                    s["step"] += 1
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As the base class's, which would cast every state tensor to its parameter's type: moments, scales and masters
        keep theirs.  The step count goes over from and to `capturable`; a captured step has to be captured again, after
        one eager step.  Moments of the other `state_bits` are refused; a missing master is made from its parameter by the
        next step."""
        moments = torch.float8_e4m3fn if self.state_bits == 8 else torch.float32
        if any(state["exp_avg"].dtype != moments for state in state_dict["state"].values() if "exp_avg" in state):
            raise ValueError(f"the saved moments are not those of state_bits={self.state_bits}")
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            steps = group.pop("step_tensor", None)
            group.pop("lr_tensor", None)
            for i, p in zip(saved["params"], group["params"]):
                for key, value in state_dict["state"].get(i, {}).items():
                    if isinstance(value, torch.Tensor):
                        self.state[p][key] = value.detach().to(device=p.device, copy=True)
                if self.state.get(p):
                    if steps is not None:
                        self.state[p]["step"] = int(steps)
                    if not self.master:
                        self.state[p].pop("master", None)
