"""Tensor-level wrappers over the C ABI (include/hdcmamba_b200.h).

Each op validates device / dtype / layout, allocates its outputs through the torch
caching allocator on the current stream, and launches through ``_lib.call``.
Only CUDA tensors are accepted: there is no CPU path.
"""
import ctypes
import functools

import torch

from . import _lib

try:  # the stream's address without a Stream object (0.2 us for 2.3)
    from torch._C import _cuda_getCurrentRawStream as _current_raw_stream
except ImportError:  # pragma: no cover
    def _current_raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream

_DT = {torch.float32: _lib.HDC_F32, torch.bfloat16: _lib.HDC_BF16}


def _code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"hdcmamba_b200: unsupported dtype {t.dtype} (float32 or bfloat16)") from None


def _cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("hdcmamba_b200 kernels run on CUDA tensors only (got a CPU tensor)")


def _stream(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _same_dtype(ref, *ts):
    for t in ts:
        if t is not None and t.dtype != ref.dtype:
            raise TypeError(f"hdcmamba_b200: dtype mismatch ({t.dtype} vs {ref.dtype})")


def check_device():
    """Synchronise the current device and raise HdcError if a bounded wait inside a kernel has run
    out since the last check (the error is cleared): the outputs of the call that waited are
    invalid.  Kernels report such a wait on the device only, so a training loop calls this once
    in a while (say with each checkpoint)."""
    torch.cuda.synchronize()
    code = _lib.load().hdc_device_error(1)
    if code != 0:
        raise _lib.HdcError(f"a bounded wait inside a kernel has run out (code {code}); the outputs of that call are invalid")


# ------------------------------------------------------------------ LN + conv
def ln_conv(x, norm_w, norm_b, conv_w, conv_b, eps=1e-5, act="none", halo=None, stats=False, halo_flag=None):
    """LayerNorm + causal depthwise conv1d (width 4), optional SiLU.

    Replaces ``_fused_norm_conv_fwd_kernel`` (hdcmamba/model.py:22-72).
    x: [B, L, D]; conv_w: [D, 4] or [D, 1, 4]; halo: optional [B, 3, D].
    halo_flag: optional (flag address, generation address) of device uint32s: the CTAs that
    read the halo wait until the flag reaches the generation (a halo stored by another GPU).
    Returns out (and bf16 mean, rstd [B, L] if ``stats``)."""
    _cuda(x, norm_w, norm_b, conv_w, conv_b, halo)
    B, L, D = x.shape
    x = x.contiguous()
    nw, nb = norm_w.to(x.dtype).contiguous(), norm_b.to(x.dtype).contiguous()
    cw = conv_w.reshape(D, 4).to(x.dtype).contiguous()
    cb = conv_b.to(x.dtype).contiguous()
    if halo is not None:
        halo = halo.to(x.dtype).contiguous()
        if tuple(halo.shape) != (B, 3, D):
            raise ValueError(f"halo must be [B, 3, D], got {tuple(halo.shape)}")
    out = torch.empty_like(x)
    mean = rstd = None
    if stats:
        mean = torch.empty(B, L, device=x.device, dtype=torch.bfloat16)
        rstd = torch.empty(B, L, device=x.device, dtype=torch.bfloat16)
    a = {"none": _lib.HDC_ACT_NONE, "silu": _lib.HDC_ACT_SILU}[act]
    if halo_flag is not None:
        if halo is None:
            raise ValueError("halo_flag needs a halo")
        _lib.call("hdc_ln_conv_fwd_halo_flag", _code(x), _p(x), _p(nw), _p(nb), _p(cw), _p(cb), _p(halo), _p(out),
                  _p(mean), _p(rstd), B, L, D, float(eps), a, ctypes.c_void_p(halo_flag[0]),
                  ctypes.c_void_p(halo_flag[1]), _stream(x))
    else:
        _lib.call("hdc_ln_conv_fwd", _code(x), _p(x), _p(nw), _p(nb), _p(cw), _p(cb), _p(halo), _p(out),
                  _p(mean), _p(rstd), B, L, D, float(eps), a, _stream(x))
    return (out, mean, rstd) if stats else out


# ------------------------------------------------------------------ SSM scan
def ln_conv_bwd(grad_out, x, mean, rstd, norm_w, conv_w):
    """Backward of ``ln_conv`` (act="none"): the reference's FusedNormConv1dFunction.backward
    (hdcmamba/model.py:74-124, 148-166), its formulas included.  ``mean`` / ``rstd`` are the
    forward's bf16 statistics.  Returns (dx, d_norm_w, d_norm_b, d_conv_w [D, 4], d_conv_b)
    in x.dtype."""
    _cuda(grad_out, x, mean, rstd, norm_w, conv_w)
    B, L, D = x.shape
    grad_out = grad_out.contiguous()
    x = x.contiguous()
    _same_dtype(x, grad_out)
    nw = norm_w.to(x.dtype).contiguous()
    cw = conv_w.reshape(D, 4).to(x.dtype).contiguous()
    mean = mean.to(torch.bfloat16).contiguous()
    rstd = rstd.to(torch.bfloat16).contiguous()
    dx = torch.empty_like(x)
    dnw = torch.empty(D, device=x.device, dtype=x.dtype)
    dnb = torch.empty_like(dnw)
    dcw = torch.empty(D, 4, device=x.device, dtype=x.dtype)
    dcb = torch.empty_like(dnw)
    ws = torch.empty(max(int(_lib.load().hdc_ln_conv_bwd_workspace_bytes(B, L, D)), 16), device=x.device,
                     dtype=torch.uint8)
    _lib.call("hdc_ln_conv_bwd", _code(x), _p(grad_out), _p(x), _p(mean), _p(rstd), _p(nw), _p(cw), _p(dx), _p(dnw),
              _p(dnb), _p(dcw), _p(dcb), _p(ws), ws.numel(), B, L, D, _stream(x))
    return dx, dnw, dnb, dcw, dcb


def _ln_conv_params(x, *params):
    """Parameters in x's type, contiguous (conv weights [D, 4] or [D, 1, 4] as [D, 4])."""
    D = x.shape[2]
    return tuple((p.reshape(D, 4) if p.dim() > 1 else p).to(x.dtype).contiguous() for p in params)


def ln_conv_train(x, norm_w, norm_b, conv_w, conv_b, eps=1e-5):
    """``ln_conv`` without activation for training a layer of one's own
    (hdc_ln_conv_train_fwd): returns (out, mean, rstd), the row statistics in fp32 [B, L]."""
    _cuda(x, norm_w, norm_b, conv_w, conv_b)
    dt = _code(x)
    B, L, D = x.shape
    x = x.contiguous()
    nw, nb, cw, cb = _ln_conv_params(x, norm_w, norm_b, conv_w, conv_b)
    out = torch.empty_like(x)
    mean = torch.empty(B, L, device=x.device, dtype=torch.float32)
    rstd = torch.empty(B, L, device=x.device, dtype=torch.float32)
    _lib.call("hdc_ln_conv_train_fwd", dt, _p(x), _p(nw), _p(nb), _p(cw), _p(cb), _p(out), _p(mean), _p(rstd),
              B, L, D, float(eps), _stream(x))
    return out, mean, rstd


def ln_conv_train_bwd(grad_out, x, mean, rstd, norm_w, norm_b, conv_w):
    """The derivative of ``ln_conv_train`` (hdc_ln_conv_train_bwd), the norm bias and the rows
    before the sequence included.  Returns (dx, d_norm_w, d_norm_b, d_conv_w [D, 4], d_conv_b)
    in x.dtype."""
    _cuda(grad_out, x, mean, rstd, norm_w, norm_b, conv_w)
    dt = _code(x)
    B, L, D = x.shape
    _same_dtype(x, grad_out)
    if grad_out.shape != x.shape:
        raise ValueError(f"grad_out {list(grad_out.shape)} must have x's shape {list(x.shape)}")
    _f32_state(mean, (B, L), "mean")
    _f32_state(rstd, (B, L), "rstd")
    grad_out, x = grad_out.contiguous(), x.contiguous()
    nw, nb, cw = _ln_conv_params(x, norm_w, norm_b, conv_w)
    dx, dnw, dnb, dcw, dcb = (torch.empty_like(t) for t in (x, nw, nw, cw, nw))
    ws = torch.empty(max(int(_lib.load().hdc_ln_conv_bwd_workspace_bytes(B, L, D)), 16), device=x.device,
                     dtype=torch.uint8)
    _lib.call("hdc_ln_conv_train_bwd", dt, _p(grad_out), _p(x), _p(mean), _p(rstd), _p(nw), _p(nb), _p(cw), _p(dx),
              _p(dnw), _p(dnb), _p(dcw), _p(dcb), _p(ws), ws.numel(), B, L, D, _stream(x))
    return dx, dnw, dnb, dcw, dcb


def _row_view(t, what):
    """(batch stride, row stride) of a [B, L, cols] view whose last dim is unit-stride."""
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{what} must be a [B, L, cols] view with unit column stride")
    return t.stride(0), t.stride(1)


def ssm_chunk_stats(projs, A_log, d_state, chunk, out=None):
    """Per-chunk statistics [B, N, 2*ds] fp32 (last state, summed log decay), bf16-rounded.

    Replaces the last_state / chunk_decay outputs of ``_ssm_intra_v2`` (hdcmamba/model.py:175-198).
    ``out``: optional contiguous fp32 [B, N, 2*ds] tensor to write into."""
    _cuda(projs, A_log, out)
    B, L, P = projs.shape
    if P < 3 * d_state or L % chunk != 0:
        raise ValueError(f"projs [B, L, {P}] needs >= 3*d_state columns and L % chunk == 0")
    sb, st = _row_view(projs, "projs")
    a = A_log.to(projs.dtype).contiguous()
    shape = (B, L // chunk, 2 * d_state)
    if out is not None and (tuple(out.shape) != shape or out.dtype != torch.float32 or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous fp32 {list(shape)} tensor")
    stats = out if out is not None else torch.empty(shape, device=projs.device, dtype=torch.float32)
    _lib.call("hdc_ssm_chunk_stats", _code(projs), _p(projs), sb, st, _p(a), _p(stats), B, L, d_state, chunk,
              _stream(projs))
    return stats


def ssm_scan_out(projs, A_log, stats, n_prev, d_state, chunk, out=None):
    """Outputs of the chunked scan given chunk statistics of [0, n_prev + N) chunks.

    Replaces ``_ssm_scan_v2`` + ``_ssm_inter_v2`` (hdcmamba/model.py:200-233).
    ``out``: optional [B, L, >=ds] view (unit column stride) to write into."""
    _cuda(projs, A_log, stats, out)
    B, L, P = projs.shape
    if P < 3 * d_state or L % chunk != 0:
        raise ValueError(f"projs [B, L, {P}] needs >= 3*d_state columns and L % chunk == 0")
    sb, st = _row_view(projs, "projs")
    a = A_log.to(projs.dtype).contiguous()
    if out is None:
        out = torch.empty(B, L, d_state, device=projs.device, dtype=projs.dtype)
    _same_dtype(projs, out)
    osb, ost = _row_view(out, "out")
    stats = stats.contiguous()
    if stats.dtype != torch.float32 or stats.shape[0] != B or stats.shape[1] != n_prev + L // chunk:
        raise ValueError("stats must be fp32 [B, n_prev + L/chunk, 2*d_state]")
    _lib.call("hdc_ssm_scan_out", _code(projs), _p(projs), sb, st, _p(a), _p(stats), stats.stride(0), n_prev,
              _p(out), osb, ost, B, L, d_state, chunk, _stream(projs))
    return out


def ssm_scan_out_blocked(projs, A_log, stats, stats_sb, block_chunks, block_stride, n_prev, d_state, chunk,
                         out=None, wait=None):
    """ssm_scan_out reading the statistics of chunks [0, n_prev + N) in place from a
    rank-major gathered buffer: ``stats`` is a 1-D fp32 tensor whose element 0 is chunk 0
    of block 0; chunk m of batch b is at (m // block_chunks) * block_stride + b * stats_sb
    + (m % block_chunks) * 2 * ds (hdc_ssm_scan_out_blocked).  ``wait``: optional
    (flags address, mask, generation address): the kernel waits for the flags before it
    reads statistics stored by other GPUs."""
    _cuda(projs, A_log, stats, out)
    B, L, P = projs.shape
    if P < 3 * d_state or L % chunk != 0:
        raise ValueError(f"projs [B, L, {P}] needs >= 3*d_state columns and L % chunk == 0")
    if stats.dtype != torch.float32 or stats.dim() != 1 or stats.stride(0) != 1:
        raise ValueError("stats must be a 1-D contiguous fp32 tensor")
    m_end = n_prev + L // chunk
    last_blk = (m_end - 1) // block_chunks
    rows_in_last = m_end - last_blk * block_chunks
    need = last_blk * block_stride + (B - 1) * stats_sb + rows_in_last * 2 * d_state
    if need > stats.numel():
        raise ValueError(f"stats holds {stats.numel()} floats, the layout reads up to {need}")
    sb, st = _row_view(projs, "projs")
    a = A_log.to(projs.dtype).contiguous()
    if out is None:
        out = torch.empty(B, L, d_state, device=projs.device, dtype=projs.dtype)
    _same_dtype(projs, out)
    osb, ost = _row_view(out, "out")
    wf, wm, wg = wait if wait is not None else (0, 0, 0)
    _lib.call("hdc_ssm_scan_out_blocked", _code(projs), _p(projs), sb, st, _p(a), _p(stats), stats_sb, block_chunks,
              block_stride, n_prev, _p(out), osb, ost, B, L, d_state, chunk, ctypes.c_void_p(wf), wm,
              ctypes.c_void_p(wg), _stream(projs))
    return out


def ssm_scan(projs, A_log, d_state, chunk, out=None):
    """The whole diagonal-SSM chunked scan (hdcmamba/model.py:175-233, launched 345-363):
    ``hdc_ssm_scan_fwd``, statistics then outputs, enqueued back to back.
    ``out``: optional [B, L, >=ds] view (unit column stride) to write into."""
    _cuda(projs, A_log, out)
    B, L, P = projs.shape
    if P < 3 * d_state or L % chunk != 0:
        raise ValueError(f"projs [B, L, {P}] needs >= 3*d_state columns and L % chunk == 0")
    sb, st = _row_view(projs, "projs")
    a = A_log.to(projs.dtype).contiguous()
    if out is None:
        out = torch.empty(B, L, d_state, device=projs.device, dtype=projs.dtype)
    _same_dtype(projs, out)
    osb, ost = _row_view(out, "out")
    stats = torch.empty(B, L // chunk, 2 * d_state, device=projs.device, dtype=torch.float32)
    _lib.call("hdc_ssm_scan_fwd", _code(projs), _p(projs), sb, st, _p(a), _p(stats), _p(out), osb, ost, B, L,
              d_state, chunk, _stream(projs))
    return out


# ------------------------------------------------------------------ slot scan
def slot_workspace_bytes(B, L, H, hd, chunk):
    return int(_lib.load().hdc_slot_workspace_bytes(B, L, H, hd, chunk))


def feature_block(hd):
    b = 1
    while b < hd:
        b <<= 1
    return max(64, b)


_SLOT_PATHS = {"auto": 0, "simt": 1, "tc": 2}


def slot_scan(q, k, v, num_heads, chunk, gamma=None, log_a=None, rows=None, y=None, y_strides=None,
              state_in=None, return_state=False, path="auto", path_used=None):
    """Slot memory scan (replaces ``_slot_all_fused``, hdcmamba/model.py:236-272).

    q, k, v: [B, L, H*hd] views sharing strides (unit last-dim stride), raw
    (before phi).  gamma: [H] (in the activation dtype) or log_a: fp32 [B, L, H].
    y: optional output tensor with element strides ``y_strides = (sb, sh, st)``
    (element (b, t, h, d) at b*sb + h*sh + t*st + d); default [B, L, H, hd].
    path: "auto", "simt" (CUDA-core kernel) or "tc" (tcgen05 required, error otherwise);
    ``path_used`` (a list) receives "tc" or "simt".
    Returns y (and the fp32 final state [B, H, bd, bd] if ``return_state``)."""
    _cuda(q, k, v, gamma, log_a, y, state_in)
    if path not in _SLOT_PATHS:
        raise ValueError(f"path must be one of {sorted(_SLOT_PATHS)}")
    _same_dtype(q, k, v)
    B, L, W = q.shape
    H = num_heads
    hd = W // H
    if W != H * hd or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must be [B, L, H*hd] with equal shapes")
    if q.stride() != k.stride() or q.stride() != v.stride() or q.stride(2) != 1:
        raise ValueError("q, k, v must share strides with unit last-dim stride")
    if (gamma is None) == (log_a is None):
        raise ValueError("give exactly one of gamma (constant decay) or log_a (per-step decay)")
    if gamma is not None:
        gamma = gamma.to(q.dtype).contiguous()
    if log_a is not None:
        log_a = log_a.float().contiguous()
        if tuple(log_a.shape) != (B, L, H):
            raise ValueError("log_a must be [B, L, H]")
    rows = chunk if rows is None else rows
    if y is None:
        y = torch.empty(B, L, H, hd, device=q.device, dtype=q.dtype)
        y_strides = (L * H * hd, hd, H * hd)
    elif y_strides is None:
        raise ValueError("y_strides is required with y")
    _same_dtype(q, y)
    bd = feature_block(hd)
    state_out = torch.empty(B, H, bd, bd, device=q.device, dtype=torch.float32) if return_state else None
    if state_in is not None:
        state_in = state_in.float().contiguous()
    nbytes = slot_workspace_bytes(B, L, H, hd, chunk)
    ws = torch.empty(max(nbytes, 16), device=q.device, dtype=torch.uint8)
    used = ctypes.c_int(-1)
    _lib.call("hdc_slot_scan_fwd_path", _code(q), _p(q), _p(k), _p(v), q.stride(0), q.stride(1), _p(gamma),
              _p(log_a), _p(y), y_strides[0], y_strides[1], y_strides[2], _p(state_in), _p(state_out), _p(ws),
              ws.numel(), B, L, H, hd, chunk, rows, _SLOT_PATHS[path], ctypes.byref(used), _stream(q))
    if path_used is not None:
        path_used.append("tc" if used.value == 1 else "simt")
    return (y, state_out) if return_state else y


def slot_gate_supported(q, num_heads, chunk):
    """True when hdc_slot_gate_fwd (tcgen05, fused gate epilogue) accepts these inputs."""
    B, L, W = q.shape
    hd = W // num_heads
    return (q.dtype == torch.bfloat16 and hd <= 64 and hd % 8 == 0 and W >= 64 and chunk in (64, 128, 256)
            and L % chunk == 0 and q.stride(2) == 1 and q.stride(1) % 8 == 0 and q.data_ptr() % 16 == 0)


def slot_scan_gate(q, k, v, num_heads, chunk, gate, gn_w, gn_b, out, out_strides, gamma=None, log_a=None,
                   state_in=None, return_state=False):
    """Slot scan with GroupNorm(head) * sigmoid(gate) fused into its epilogue
    (replaces ``_slot_all_fused`` plus the slot half of ``_fused_gnorm_gate_cat_kernel``,
    hdcmamba/model.py:236-293).  gate: [B, L, H*hd] view (unit last stride); out:
    tensor with element strides ``out_strides = (sb, sh, st)``."""
    _cuda(q, k, v, gamma, log_a, gate, gn_w, gn_b, out, state_in)
    _same_dtype(q, k, v, gate, out)
    B, L, W = q.shape
    H = num_heads
    hd = W // H
    if q.stride() != k.stride() or q.stride() != v.stride() or gate.stride(2) != 1:
        raise ValueError("q, k, v must share strides; gate needs a unit last stride")
    if (gamma is None) == (log_a is None):
        raise ValueError("give exactly one of gamma or log_a")
    if gamma is not None:
        gamma = gamma.to(q.dtype).contiguous()
    if log_a is not None:
        log_a = log_a.float().contiguous()
    gw = gn_w.to(q.dtype).contiguous()
    gb = gn_b.to(q.dtype).contiguous()
    bd = feature_block(hd)
    state_out = torch.empty(B, H, bd, bd, device=q.device, dtype=torch.float32) if return_state else None
    if state_in is not None:
        state_in = state_in.float().contiguous()
    ws = torch.empty(max(slot_workspace_bytes(B, L, H, hd, chunk), 16), device=q.device, dtype=torch.uint8)
    _lib.call("hdc_slot_gate_fwd", _code(q), _p(q), _p(k), _p(v), q.stride(0), q.stride(1), _p(gamma), _p(log_a),
              _p(gate), gate.stride(0), gate.stride(1), _p(gw), _p(gb), _p(out), out_strides[0], out_strides[1],
              out_strides[2], _p(state_in), _p(state_out), _p(ws), ws.numel(), B, L, H, hd, chunk, _stream(q))
    return (out, state_out) if return_state else out


def slot_workspace(B, L, num_heads, head_dim, chunk, device):
    """A device workspace for one slot call of this shape (uint8)."""
    return torch.empty(max(slot_workspace_bytes(B, L, num_heads, head_dim, chunk), 16), device=device,
                       dtype=torch.uint8)


def _f32_out(t, shape, what):
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != torch.float32 or not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous fp32 {list(shape)} tensor")


def slot_state(k, v, num_heads, chunk, gamma=None, log_a=None, state_out=None, decay_out=None, workspace=None):
    """State after the whole sequence from a zero start, fp32 [B, H, 64, 64], and the
    product of all chunk decays [B, H] (for sequence-parallel carries).  ``workspace``
    (from ``slot_workspace``) keeps the segment states for ``slot_scan_gate_carry``."""
    _cuda(k, v, gamma, log_a, state_out, decay_out, workspace)
    _same_dtype(k, v)
    B, L, W = k.shape
    H = num_heads
    hd = W // H
    if k.stride() != v.stride() or k.stride(2) != 1:
        raise ValueError("k, v must share strides with unit last-dim stride")
    if gamma is not None:
        gamma = gamma.to(k.dtype).contiguous()
    if log_a is not None:
        log_a = log_a.float().contiguous()
    _f32_out(state_out, (B, H, 64, 64), "state_out")
    _f32_out(decay_out, (B, H), "decay_out")
    state = state_out if state_out is not None else torch.empty(B, H, 64, 64, device=k.device, dtype=torch.float32)
    decay = decay_out if decay_out is not None else torch.empty(B, H, device=k.device, dtype=torch.float32)
    ws = workspace if workspace is not None else slot_workspace(B, L, H, hd, chunk, k.device)
    _lib.call("hdc_slot_state_fwd", _code(k), _p(k), _p(v), k.stride(0), k.stride(1), _p(gamma), _p(log_a),
              _p(state), _p(decay), _p(ws), ws.numel(), B, L, H, hd, chunk, _stream(k))
    return state, decay


def slot_scan_gate_carry(q, k, v, num_heads, chunk, gate, gn_w, gn_b, out, out_strides, prev_state, prev_decay,
                         prev_stride, n_prev, workspace, gamma=None, log_a=None, wait=None):
    """``slot_scan_gate`` for one rank's part of the sequence (hdc_slot_gate_carry_fwd):
    the entering state folds the n_prev earlier parts, part s with its fp32 state at
    prev_state[s*prev_stride:] ([B, H, 64, 64]) and decay at prev_decay[s*prev_stride:]
    ([B, H]); ``workspace`` is the one ``slot_state`` filled for the same k, v.  ``wait``:
    optional (flags address, mask, generation address): the kernel waits for the flags
    before it reads earlier parts stored by other GPUs."""
    _cuda(q, k, v, gamma, log_a, gate, gn_w, gn_b, out, prev_state, prev_decay, workspace)
    _same_dtype(q, k, v, gate, out)
    B, L, W = q.shape
    H = num_heads
    hd = W // H
    if q.stride() != k.stride() or q.stride() != v.stride() or gate.stride(2) != 1:
        raise ValueError("q, k, v must share strides; gate needs a unit last stride")
    if (gamma is None) == (log_a is None):
        raise ValueError("give exactly one of gamma or log_a")
    if n_prev > 0:
        if prev_state.data_ptr() % 16 != 0 or prev_stride % 4 != 0:
            raise ValueError("prev_state must be 16-byte aligned and prev_stride a multiple of 4")
        for t, per in ((prev_state, B * H * 4096), (prev_decay, B * H)):
            if t.dtype != torch.float32 or t.dim() != 1 or t.stride(0) != 1:
                raise ValueError("prev_state / prev_decay must be 1-D contiguous fp32 tensors")
            if (n_prev - 1) * prev_stride + per > t.numel():
                raise ValueError("prev_state / prev_decay too short for n_prev parts")
    if gamma is not None:
        gamma = gamma.to(q.dtype).contiguous()
    if log_a is not None:
        log_a = log_a.float().contiguous()
    gw = gn_w.to(q.dtype).contiguous()
    gb = gn_b.to(q.dtype).contiguous()
    _lib.call("hdc_slot_gate_carry_fwd", _code(q), _p(q), _p(k), _p(v), q.stride(0), q.stride(1), _p(gamma),
              _p(log_a), _p(gate), gate.stride(0), gate.stride(1), _p(gw), _p(gb), _p(out), out_strides[0],
              out_strides[1], out_strides[2], _p(prev_state if n_prev else None), _p(prev_decay if n_prev else None),
              prev_stride, n_prev, None, _p(workspace), workspace.numel(), B, L, H, hd, chunk,
              ctypes.c_void_p(wait[0] if wait else 0), wait[1] if wait else 0, ctypes.c_void_p(wait[2] if wait else 0),
              _stream(q))
    return out


# ------------------------------------------------------------------ gate / concat / LN
def gate_cat(y_slot, slot_strides, slot_rows, y_ssm, ssm_strides, gate, gate_strides, gn_w, gn_b, out,
             out_strides, B, L, H, hd, ds):
    """GroupNorm(head) * sigmoid(gate), concatenated after y_ssm (replaces
    ``_fused_gnorm_gate_cat_kernel``, hdcmamba/model.py:274-295).  Strides are in
    elements and follow the reference launch (hdcmamba/model.py:377); the
    pointers are the base addresses of the given tensors (views allowed)."""
    _cuda(y_slot, y_ssm, gate, gn_w, gn_b, out)
    _same_dtype(out, y_slot, y_ssm, gate)
    gw = gn_w.to(out.dtype).contiguous()
    gb = gn_b.to(out.dtype).contiguous()
    _lib.call("hdc_gate_cat_fwd", _code(out), _p(y_slot), slot_strides[0], slot_strides[1], slot_strides[2],
              slot_rows, _p(y_ssm), ssm_strides[0], ssm_strides[1], _p(gate), gate_strides[0], gate_strides[1],
              _p(gw), _p(gb), _p(out), out_strides[0], out_strides[1], B, L, H, hd, ds, _stream(out))
    return out


def row_layernorm(x, eps=1e-5, out=None):
    """LayerNorm over the last dim without affine, fp32 statistics, result in x.dtype
    (replaces ``F.layer_norm(combined.float(), (ds+dm,)).to(x.dtype)``, hdcmamba/model.py:382)."""
    _cuda(x, out)
    if not x.is_contiguous():
        raise ValueError("row_layernorm needs a contiguous input")
    if out is None:
        out = torch.empty_like(x)
    width = x.shape[-1]
    _lib.call("hdc_row_layernorm", _code(x), _p(x), _p(out), x.numel() // width, width, float(eps), _stream(x))
    return out


def layer_norm(x, weight, bias, eps=1e-5, out=None):
    """nn.LayerNorm over the last dim with its elementwise affine: fp32 statistics and
    affine, result in x.dtype (hdc_row_layernorm_affine; replaces the final norms,
    hdcmamba/model.py:400, 404 and train.py:121, 135)."""
    _cuda(x, weight, bias, out)
    if not x.is_contiguous():
        raise ValueError("layer_norm needs a contiguous input")
    if out is None:
        out = torch.empty_like(x)
    width = x.shape[-1]
    w, b = weight.to(x.dtype).contiguous(), bias.to(x.dtype).contiguous()
    _lib.call("hdc_row_layernorm_affine", _code(x), _p(x), _p(w), _p(b), _p(out), x.numel() // width, width,
              float(eps), _stream(x))
    return out


# ------------------------------------------------------------------ single-token decode
def ln_conv_step(x, norm_w, norm_b, conv_w, conv_b, window, eps=1e-5, out=None):
    """LN + conv of one new row per sequence, x [B, D]; ``window`` fp32 [B, 3, D] (the
    normalised rows t-3..t-1) is shifted in place (hdc_ln_conv_step)."""
    _cuda(x, norm_w, norm_b, conv_w, conv_b, window, out)
    B, D = x.shape
    x = x.contiguous()
    if window.dtype != torch.float32 or tuple(window.shape) != (B, 3, D) or not window.is_contiguous():
        raise ValueError(f"window must be a contiguous fp32 [{B}, 3, {D}] tensor")
    dt = x.dtype
    out = torch.empty_like(x) if out is None else out
    _lib.call("hdc_ln_conv_step", _code(x), _p(x), _p(norm_w.to(dt).contiguous()), _p(norm_b.to(dt).contiguous()),
              _p(conv_w.reshape(D, 4).to(dt).contiguous()), _p(conv_b.to(dt).contiguous()), _p(window), _p(out), B, D,
              float(eps), _stream(x))
    return out


def ssm_step(projs, A_log, h, cum, G, d_state, pos, chunk, out):
    """One diagonal-SSM step for rows projs [B, P]; h / cum / G fp32 [B, ds] updated in
    place; ``pos`` a device int32 tensor holding the row index within the chunk (the chunk
    is folded into G at row chunk-1); writes out [B, >=ds] (unit column stride)."""
    _cuda(projs, A_log, h, cum, G, out, pos)
    B = projs.shape[0]
    if projs.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("projs / out need a unit column stride")
    a = A_log.to(projs.dtype).contiguous()
    _lib.call("hdc_ssm_step", _code(projs), _p(projs), projs.stride(0), _p(a), _p(h), _p(cum), _p(G), _p(out),
              out.stride(0), B, d_state, _p(pos), chunk, _stream(projs))
    return out


def ssm_carry(stats, dtype):
    """Carry G [B, ds] fp32 after the chunks of ``stats`` [B, N, 2ds] (hdc_ssm_carry_fwd);
    ``dtype`` is the activation dtype (selects the exp of that prefill path)."""
    _cuda(stats)
    B, N, two_ds = stats.shape
    G = torch.empty(B, two_ds // 2, device=stats.device, dtype=torch.float32)
    code = 1 if dtype == torch.bfloat16 else 0
    _lib.call("hdc_ssm_carry_fwd", code, _p(stats.contiguous()), B, N, two_ds // 2, _p(G), _stream(stats))
    return G


def slot_step(q, k, v, gate, num_heads, gamma, gn_w, gn_b, R, U, k_cache, v_cache, out, pos):
    """The next row (index in the device int32 ``pos``) of the current chunk of the slot
    scan with GroupNorm(head) * sigmoid(gate) (hdc_slot_step).  q / k / v / gate: [B, H*hd] views sharing one batch stride; R / U fp32
    [B, H, 64, 64]; k_cache / v_cache [B, H, C, 64]; out [B, H*hd] view (unit column stride)."""
    _cuda(q, k, v, gate, gamma, gn_w, gn_b, R, U, k_cache, v_cache, out, pos)
    B, W = q.shape
    H = num_heads
    hd = W // H
    C = k_cache.shape[2]
    if not (q.stride() == k.stride() == v.stride() == gate.stride()) or q.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("q / k / v / gate must share strides with unit column stride")
    dt = q.dtype
    _lib.call("hdc_slot_step", _code(q), _p(q), _p(k), _p(v), _p(gate), q.stride(0), _p(gamma.to(dt).contiguous()),
              _p(gn_w.to(dt).contiguous()), _p(gn_b.to(dt).contiguous()), _p(R), _p(U), _p(k_cache), _p(v_cache),
              _p(out), out.stride(0), B, H, hd, C, _p(pos), _stream(q))
    return out


# ------------------------------------------------------------------ gated recurrence
@functools.lru_cache(maxsize=4096)
def _size(name, *sizes):
    """A size that the library computes from sizes alone."""
    return int(getattr(_lib.load(), name)(*sizes))


def _raw_stream(t):
    """The current stream of t's device as an int."""
    return _current_raw_stream(t.device.index)


def _a(t):
    """A tensor's address as a plain int (ctypes converts it), None for none."""
    return t.data_ptr() if t is not None else None


_ACTS = {"none": _lib.HDC_ACT_NONE, "silu": _lib.HDC_ACT_SILU}


def _workspace(nbytes, device):
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def _f32_state(t, shape, what):
    if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous fp32 {list(shape)} tensor")


def _gated_args(projs, A_log, d_state, reset, rows):
    """Checks shared by the gated-recurrence ops; A_log and reset made contiguous."""
    if projs.dim() != len(rows) + 1 or projs.shape[-1] < 3 * d_state or d_state < 1:
        raise ValueError(f"projs {list(projs.shape)} must be {list(rows)} rows of >= 3*d_state columns")
    if projs.shape[-1] > 1 and projs.stride(-1) != 1:
        raise ValueError("projs needs a unit column stride")
    if A_log.shape != (d_state,):
        raise ValueError(f"A_log must be [{d_state}], got {list(A_log.shape)}")
    if reset is not None:
        if reset.dtype not in (torch.bool, torch.uint8) or reset.shape != rows:
            raise ValueError(f"reset must be a bool {list(rows)} tensor")
        reset = reset.contiguous()
    return A_log.contiguous(), reset


def gated_scan(projs, A_log, d_state, h0=None, reset=None, out=None, return_states=False):
    """Gated linear recurrence over whole sequences (hdc_gated_scan_fwd): the Block's SSM gates
    (hdcmamba/model.py:189-193) with no chunk rounding, h_t = exp(d A) h_{t-1} + d b x with
    d = softplus(dt), A = -exp(A_log).

    projs: [B, L, >=3*d_state] view (unit column stride), columns dt | x | b; L may be 0.
    h0: optional fp32 [B, d_state] state before the first step.  reset: optional bool [B, L];
    a true step starts from a zero state.  out: optional [B, L, d_state] view (unit column
    stride).  Returns (y in projs.dtype, h_last fp32 [B, d_state]) and, if ``return_states``,
    the states that ``gated_scan_bwd`` needs.  For autograd use ``recurrent.gated_scan``.
    Waits between the tiles of a sequence are bounded: see ``check_device``."""
    _cuda(projs, A_log, h0, reset, out)
    dt = _code(projs)
    if projs.dim() != 3:
        raise ValueError("projs must be [B, L, cols]")
    B, L, _ = projs.shape
    A_log, reset = _gated_args(projs, A_log, d_state, reset, (B, L))
    if h0 is not None:
        h0 = h0.float().contiguous()
        if h0.shape != (B, d_state):
            raise ValueError(f"h0 must be [{B}, {d_state}]")
    if out is None:
        out = torch.empty(B, L, d_state, device=projs.device, dtype=projs.dtype)
    else:
        _same_dtype(projs, out)
        if out.shape != (B, L, d_state) or (d_state > 1 and out.stride(2) != 1):
            raise ValueError(f"out must be a [{B}, {L}, {d_state}] view with unit column stride")
    h_last = torch.empty(B, d_state, device=projs.device, dtype=torch.float32)
    states = None
    if return_states:
        rows = _size("hdc_gated_scan_state_rows")
        states = torch.empty(B, (L + rows - 1) // rows, d_state, device=projs.device, dtype=torch.float32)
    ws = _workspace(_size("hdc_gated_scan_workspace_bytes", B, L, d_state), projs.device)
    _lib.call("hdc_gated_scan_fwd", dt, _code(A_log), _a(projs), projs.stride(0), projs.stride(1), _a(A_log), _a(h0),
              _a(reset), _a(out), out.stride(0), out.stride(1), _a(h_last), _a(states), _a(ws),
              ws.numel() if ws is not None else 0, B, L, d_state, _raw_stream(projs))
    return (out, h_last, states) if return_states else (out, h_last)


def gated_scan_bwd(dy, projs, A_log, states, d_state, reset=None, dh_last=None, need_dh0=False, out=None):
    """Gradient of ``gated_scan`` (hdc_gated_scan_bwd).  ``states`` as returned by the forward
    on the same inputs; dy: [B, L, d_state] view (unit column stride) in projs.dtype; dh_last:
    optional fp32 [B, d_state].  out: optional [B, L, >=3*d_state] view that receives dprojs
    (its first 3*d_state columns).  Returns (dprojs, dA_log in A_log.dtype, dh0 fp32
    [B, d_state] or None)."""
    _cuda(dy, projs, A_log, states, reset, dh_last, out)
    if projs.dim() != 3:
        raise ValueError("projs must be [B, L, cols]")
    B, L, _ = projs.shape
    A_log, reset = _gated_args(projs, A_log, d_state, reset, (B, L))
    _same_dtype(projs, dy)
    if dy.shape != (B, L, d_state):
        raise ValueError(f"dy must be [{B}, {L}, {d_state}]")
    rows = _size("hdc_gated_scan_state_rows")
    _f32_state(states, (B, (L + rows - 1) // rows, d_state), "states")
    if dh_last is not None:
        dh_last = dh_last.float().contiguous()
        if dh_last.shape != (B, d_state):
            raise ValueError(f"dh_last must be [{B}, {d_state}]")
    if out is not None:
        _same_dtype(projs, out)
        if out.dim() != 3 or out.shape[:2] != (B, L) or out.shape[2] < 3 * d_state or out.stride(2) != 1:
            raise ValueError(f"out must be a [{B}, {L}, >= {3 * d_state}] view with unit column stride")
    return _gated_scan_bwd(dy, projs, A_log, states, d_state, reset, dh_last, need_dh0, out)


def _gated_scan_bwd(dy, projs, A_log, states, d_state, reset, dh_last, need_dh0, out):
    """``gated_scan_bwd`` on arguments that have been checked (A_log, reset, dh_last contiguous)."""
    B, L, _ = projs.shape
    dev = projs.device
    if d_state > 1 and dy.stride(2) != 1:
        dy = dy.contiguous()
    if out is None:
        out = torch.empty(B, L, 3 * d_state, device=dev, dtype=projs.dtype)
    dA = torch.empty_like(A_log)
    dh0 = torch.empty(B, d_state, device=dev, dtype=torch.float32) if need_dh0 else None
    nbytes = _size("hdc_gated_scan_bwd_workspace_bytes", B, L, d_state)
    ws = _workspace(nbytes, dev)
    _lib.call("hdc_gated_scan_bwd", _code(projs), _code(A_log), _a(projs), projs.stride(0), projs.stride(1), _a(A_log),
              _a(states), _a(reset), _a(dy), dy.stride(0), dy.stride(1), _a(dh_last), _a(out), out.stride(0),
              out.stride(1), _a(dA), _a(dh0), _a(ws), nbytes, B, L, d_state, _raw_stream(projs))
    return out, dA, dh0


def gated_step(projs, A_log, h, d_state, reset=None, out=None, h_out=None):
    """One step of ``gated_scan`` per sequence (hdc_gated_step): projs [B, >=3*d_state] (unit
    column stride), h fp32 [B, d_state], updated in place unless ``h_out`` is given; reset:
    optional bool [B].  Returns (y [B, d_state] in projs.dtype, the new state)."""
    _cuda(projs, A_log, h, reset, out, h_out)
    dt = _code(projs)
    if projs.dim() != 2:
        raise ValueError("projs must be [B, cols]")
    B = projs.shape[0]
    A_log, reset = _gated_args(projs, A_log, d_state, reset, (B,))
    _f32_state(h, (B, d_state), "h")
    if h_out is None:
        h_out = h
    else:
        _f32_state(h_out, (B, d_state), "h_out")
    if out is None:
        out = torch.empty(B, d_state, device=projs.device, dtype=projs.dtype)
    else:
        _same_dtype(projs, out)
        if out.shape != (B, d_state) or (d_state > 1 and out.stride(1) != 1):
            raise ValueError(f"out must be a [{B}, {d_state}] view with unit column stride")
    _lib.call("hdc_gated_step", dt, _code(A_log), _a(projs), projs.stride(0), _a(A_log), _a(h), _a(reset), _a(h_out),
              _a(out), out.stride(0), B, d_state, _raw_stream(projs))
    return out, h_out


# ------------------------------------------------------------------ group norm + activation
def _positions(x):
    """x [N, ..., C] as a [N, S, C] view with unit channel stride (a copy only when the
    strides of the positions do not allow one)."""
    if x.dim() < 2:
        raise ValueError(f"group_norm_act needs [N, ..., C], got {list(x.shape)}")
    if x.dim() != 3:
        S = 1
        for n in x.shape[1:-1]:
            S *= n
        x = x.reshape(x.shape[0], S, x.shape[-1])
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _norm_params(x, num_groups, weight, bias):
    C = x.shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups != 0:
        raise ValueError(f"{C} channels do not split into {num_groups} groups")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is not None and t.shape != (C,):
            raise ValueError(f"{what} must be [{C}], got {list(t.shape)}")
    if weight is not None and bias is not None:
        _same_dtype(weight, bias)
    ref = weight if weight is not None else bias
    return (_code(ref) if ref is not None else _code(x), weight.contiguous() if weight is not None else None,
            bias.contiguous() if bias is not None else None)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", stats=False):
    """Group norm with an activation, channels last (hdc_group_norm_fwd): x [N, ..., C],
    statistics of each sample and group of C / num_groups neighbouring channels over all
    positions in between ([N, C]: over the group's channels alone, as the Block's GroupNorm
    per head and token, hdcmamba/model.py:285-292).  act: "none" or "silu".  Returns y (and
    fp32 mean, rstd [N, num_groups] if ``stats``).  For autograd use
    ``recurrent.group_norm_act``."""
    _cuda(x, weight, bias)
    dt = _code(x)
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}")
    x3 = _positions(x)
    pd, weight, bias = _norm_params(x, num_groups, weight, bias)
    N, S, C = x3.shape
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean = rstd = None
    if stats:
        mean = torch.empty(N, num_groups, device=x.device, dtype=torch.float32)
        rstd = torch.empty(N, num_groups, device=x.device, dtype=torch.float32)
    ws = _workspace(_size("hdc_group_norm_workspace_bytes", N, S, C, num_groups), x.device)
    _lib.call("hdc_group_norm_fwd", dt, pd, _a(x3), x3.stride(0), x3.stride(1), _a(weight), _a(bias), _a(y), S * C, C,
              _a(mean), _a(rstd), _a(ws), ws.numel() if ws is not None else 0, N, S, C, num_groups, float(eps),
              _ACTS[act], _raw_stream(x))
    return (y, mean, rstd) if stats else y


def group_norm_act_bwd(dy, x, mean, rstd, num_groups, weight=None, bias=None, act="none", need_params=True):
    """Gradient of ``group_norm_act`` (hdc_group_norm_bwd) from the forward's mean and rstd.
    Returns (dx in x.dtype, dweight, dbias in the parameters' type, None for a parameter that
    is None or when ``need_params`` is false)."""
    _cuda(dy, x, mean, rstd, weight, bias)
    _code(x)
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}")
    _same_dtype(x, dy)
    if dy.shape != x.shape:
        raise ValueError(f"dy {list(dy.shape)} must have x's shape {list(x.shape)}")
    _, weight, bias = _norm_params(x, num_groups, weight, bias)
    N = x.shape[0]
    _f32_state(mean, (N, num_groups), "mean")
    _f32_state(rstd, (N, num_groups), "rstd")
    return _group_norm_bwd(dy, x, mean, rstd, num_groups, weight, bias, act, need_params)


def _group_norm_bwd(dy, x, mean, rstd, num_groups, weight, bias, act, need_params):
    """``group_norm_act_bwd`` on arguments that have been checked (weight, bias contiguous)."""
    x3, d3 = _positions(x), _positions(dy)
    N, S, C = x3.shape
    ref = weight if weight is not None else bias if bias is not None else x
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    dw = torch.empty_like(weight) if need_params and weight is not None else None
    db = torch.empty_like(bias) if need_params and bias is not None else None
    nbytes = _size("hdc_group_norm_bwd_workspace_bytes", N, S, C, num_groups)
    ws = _workspace(nbytes, x.device)
    _lib.call("hdc_group_norm_bwd", _code(x), _code(ref), _a(d3), d3.stride(0), d3.stride(1), _a(x3), x3.stride(0),
              x3.stride(1), _a(mean), _a(rstd), _a(weight), _a(bias), _a(dx), S * C, C, _a(dw), _a(db), _a(ws), nbytes,
              N, S, C, num_groups, _ACTS[act], _raw_stream(x))
    return dx, dw, db
