"""A trainable recurrent layer and its differentiable operators.

The Block's SSM and slot kernels follow the reference's forward and have no gradient
(hdcmamba/model.py:175-295).  ``gated_scan`` and ``group_norm_act`` are the operators to
train such a layer with: the SSM's gates as one exact recurrence over the sequence, and the
GroupNorm of each head with SiLU, both with hand-written backward kernels.
``GatedRecurrentBlock`` joins them with the Block's LayerNorm + conv.  That one's gradient here
(``norm_conv1d``) is the derivative of its forward; ``fused_norm_conv1d_trainable`` keeps the
reference's formulas, which leave the norm bias and the rows before the sequence out of two
gradients (hdcmamba/model.py:74-124):

    blk = GatedRecurrentBlock(d_model=768, num_heads=12).cuda().bfloat16()
    loss = blk(x, reset=starts).float().square().mean(); loss.backward()   # training
    y, state = blk.prefill(prompt)                                         # serving
    y_t = blk.step(x_t, state)                                             # one token per sequence

There is no CPU path: CPU inputs raise.
"""
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .model import _require_cuda

__all__ = ["norm_conv1d", "gated_scan", "group_norm_act", "NormConv1dFunction", "GatedScanFunction",
           "GroupNormActFunction", "GatedRecurrentBlock", "RecurrentState"]


def _first_order_only():
    """Gradients of the gradients are not implemented: an error rather than missing terms."""
    if torch.is_grad_enabled():  # only with create_graph=True
        raise RuntimeError("hdcmamba_b200: norm_conv1d, gated_scan and group_norm_act are differentiable once (create_graph=False)")


class NormConv1dFunction(torch.autograd.Function):
    """(x, norm_w, norm_b, conv_w [D, 4], conv_b, eps) -> LayerNorm + causal depthwise conv1d
    (hdc_ln_conv_train_fwd / hdc_ln_conv_train_bwd); all in x's type."""

    @staticmethod
    def forward(ctx, x, norm_w, norm_b, conv_w, conv_b, eps):
        out, mean, rstd = ops.ln_conv_train(x, norm_w, norm_b, conv_w, conv_b, eps)
        ctx.save_for_backward(x, norm_w, norm_b, conv_w, mean, rstd)
        return out

    @staticmethod
    def backward(ctx, dy):
        _first_order_only()
        x, norm_w, norm_b, conv_w, mean, rstd = ctx.saved_tensors
        return (*ops.ln_conv_train_bwd(dy, x, mean, rstd, norm_w, norm_b, conv_w), None)


def norm_conv1d(x, norm, conv):
    """Differentiable LayerNorm + causal depthwise conv1d (width 4) of x [B, L, D] with the
    parameters of an ``nn.LayerNorm`` and an ``nn.Conv1d``; rows before the sequence are zeros
    before the norm."""
    _require_cuda(x)
    params = [p.to(x.dtype) for p in (norm.weight, norm.bias, conv.weight.squeeze(1), conv.bias)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *params)):
        return NormConv1dFunction.apply(x, *params, norm.eps)
    return ops.ln_conv(x, *params, norm.eps)


class GatedScanFunction(torch.autograd.Function):
    """(projs, A_log, h0, reset, d_state) -> (y, h_last); gradients for projs, A_log and h0
    (hdc_gated_scan_fwd / hdc_gated_scan_bwd)."""

    @staticmethod
    def forward(ctx, projs, A_log, h0, reset, d_state):
        A_log, reset = A_log.contiguous(), reset.contiguous() if reset is not None else None
        y, h_last, states = ops.gated_scan(projs, A_log, d_state, h0=h0, reset=reset, return_states=True)
        ctx.save_for_backward(projs, A_log, states, reset)
        ctx.d_state, ctx.h0_dtype = d_state, h0.dtype if h0 is not None else None
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    def backward(ctx, dy, dh_last):
        _first_order_only()
        projs, A_log, states, reset = ctx.saved_tensors
        ds = ctx.d_state
        if dy is None:
            dy = torch.zeros(*projs.shape[:2], ds, device=projs.device, dtype=projs.dtype)
        out = None
        if projs.shape[2] > 3 * ds:  # columns the recurrence does not read have a zero gradient
            out = torch.zeros(projs.shape, device=projs.device, dtype=projs.dtype)
        need_dh0 = ctx.h0_dtype is not None and ctx.needs_input_grad[2]
        if dh_last is not None:
            dh_last = dh_last.contiguous()
        # the forward has checked the arguments
        dprojs, dA, dh0 = ops._gated_scan_bwd(dy, projs, A_log, states, ds, reset, dh_last, need_dh0, out)
        return dprojs, dA, dh0.to(ctx.h0_dtype) if dh0 is not None else None, None, None


def gated_scan(projs, A_log, d_state, h0=None, reset=None):
    """Differentiable ``ops.gated_scan``: (y, h_last).  ``h0`` and ``h_last`` carry gradients,
    so a sequence can be trained window by window."""
    _require_cuda(projs)
    if torch.is_grad_enabled() and (projs.requires_grad or A_log.requires_grad or
                                    (h0 is not None and h0.requires_grad)):
        return GatedScanFunction.apply(projs, A_log, h0, reset, d_state)
    return ops.gated_scan(projs, A_log, d_state, h0=h0, reset=reset)


class GroupNormActFunction(torch.autograd.Function):
    """(x, weight, bias, num_groups, eps, act) -> y; gradients for x, weight and bias
    (hdc_group_norm_fwd / hdc_group_norm_bwd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act):
        weight = weight.contiguous() if weight is not None else None
        bias = bias.contiguous() if bias is not None else None
        y, mean, rstd = ops.group_norm_act(x, num_groups, weight, bias, eps=eps, act=act, stats=True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.num_groups, ctx.act = num_groups, act
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order_only()
        x, weight, bias, mean, rstd = ctx.saved_tensors
        # the forward has checked the arguments
        dx, dw, db = ops._group_norm_bwd(dy, x, mean, rstd, ctx.num_groups, weight, bias, ctx.act,
                                         ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return dx, dw, db, None, None, None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none"):
    """Differentiable ``ops.group_norm_act``."""
    _require_cuda(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return GroupNormActFunction.apply(x, weight, bias, num_groups, eps, act)
    return ops.group_norm_act(x, num_groups, weight, bias, eps=eps, act=act)


@dataclass
class RecurrentState:
    window: torch.Tensor  # fp32 [B, 3, d_model]: the last three normalised rows (LN + conv)
    h: torch.Tensor       # fp32 [B, d_state]


class GatedRecurrentBlock(nn.Module):
    """LN + conv -> in_proj -> gated_scan -> GroupNorm(heads) + SiLU -> out_proj + residual.

    The norm, the conv and the gates' parameters start as the Block's do
    (hdcmamba/model.py:306-327).  ``reset`` (bool [B, L], true at the first token of each
    document of a packed sequence) cuts the recurrence; the conv's window of three earlier
    rows is not cut."""

    def __init__(self, d_model=512, d_state=None, num_heads=8):
        super().__init__()
        d_state = d_model if d_state is None else d_state
        if d_state % num_heads != 0:
            raise ValueError("d_state must be a multiple of num_heads")
        self.d_model, self.d_state, self.num_heads = d_model, d_state, num_heads
        self.norm = nn.LayerNorm(d_model)
        self.conv1d = nn.Conv1d(d_model, d_model, kernel_size=4, groups=d_model, padding=3, bias=True)
        self.in_proj = nn.Linear(d_model, 3 * d_state, bias=True)
        with torch.no_grad():
            nn.init.normal_(self.conv1d.weight, std=0.02)
            self.conv1d.weight[:, 0, -1] += 1.0
            self.conv1d.bias.fill_(0.0)
            dt = torch.rand(d_state) * (0.1 - 0.001) + 0.001
            self.in_proj.bias[:d_state] = torch.log(torch.expm1(dt))
            self.in_proj.bias[d_state:].fill_(0.0)
        self.A_log = nn.Parameter(torch.log(torch.linspace(0.99, 0.9999, d_state)))
        self.group_norm = nn.GroupNorm(num_heads, d_state)
        self.out_proj = nn.Linear(d_state, d_model, bias=False)

    def _heads(self, y):
        """GroupNorm of each head and token with SiLU: y [..., d_state]."""
        gn = self.group_norm
        return group_norm_act(y.reshape(-1, self.d_state), self.num_heads, gn.weight, gn.bias, gn.eps,
                              "silu").reshape(y.shape)

    def _run(self, x, reset):
        x_conv = norm_conv1d(x, self.norm, self.conv1d)
        y, h = gated_scan(self.in_proj(x_conv), self.A_log, self.d_state, reset=reset)
        return x + self.out_proj(self._heads(y)), h

    def forward(self, x, reset=None):
        """x [B, L, d_model] -> [B, L, d_model]."""
        _require_cuda(x)
        return self._run(x, reset)[0]

    @torch.no_grad()
    def prefill(self, x, reset=None):
        """(forward(x), the state after it) for ``step``."""
        _require_cuda(x)
        y, h = self._run(x, reset)
        return y, RecurrentState(window=self._window(x), h=h)

    def _window(self, x):
        """The last three normalised rows; rows before the sequence are zeros, as the conv's
        padding is (their LayerNorm is the norm bias, hdcmamba/model.py:47-57)."""
        x3 = F.pad(x, (0, 0, 3, 0))[:, -3:].float()
        m = x3.mean(-1, keepdim=True)
        rs = torch.rsqrt(((x3 - m) ** 2).mean(-1, keepdim=True) + self.norm.eps)
        nw, nb = self.norm.weight.to(x.dtype).float(), self.norm.bias.to(x.dtype).float()
        return ((x3 - m) * rs * nw + nb).contiguous()

    @torch.no_grad()
    def step(self, x, state):
        """One token per sequence, x [B, d_model] -> [B, d_model]; ``state`` is updated in place."""
        _require_cuda(x)
        xc = ops.ln_conv_step(x, self.norm.weight, self.norm.bias, self.conv1d.weight.squeeze(1), self.conv1d.bias,
                              state.window, self.norm.eps)
        y, _ = ops.gated_step(F.linear(xc, self.in_proj.weight, self.in_proj.bias), self.A_log, state.h, self.d_state)
        return x + F.linear(self._heads(y), self.out_proj.weight)
