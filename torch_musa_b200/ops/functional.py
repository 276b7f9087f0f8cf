"""Functional forms of the fused operators (autograd included)."""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F

try:
    from torch.distributed.tensor import DTensor
except Exception:  # pragma: no cover  (torch built without distributed)
    DTensor = None


def _on_device(t: torch.Tensor) -> bool:
    return t.device.type == "blackwell"


# ------------------------------------------------------------------------- RMSNorm
def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension (fp32 statistics).

    On the device this is ``aten::_fused_rms_norm`` (one kernel forward, one backward)."""
    return F.rms_norm(x, (x.shape[-1],), weight, eps)


def rms_norm_residual(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6):
    """Fused ``h = x + residual; y = rms_norm(h)``; returns ``(y, h)`` (one pass over memory)."""
    if _on_device(x):
        y, h, _ = torch.ops.blackwell.rms_norm_residual(x, residual, weight, eps)     # differentiable (autograd in C++)
        return y, h
    h = x + residual
    return rms_norm(h, weight, eps), h


# ------------------------------------------------------------------------- BatchNorm (+residual) (+ReLU)
class _BatchNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, running_mean, running_var, residual, training, momentum, eps, relu):
        y, mean, invstd = torch.ops.blackwell.batch_norm_act(x, weight, bias, running_mean, running_var, residual,
                                                             training, momentum, eps, relu)
        ctx.relu, ctx.has_res, ctx.training = relu, residual is not None, training
        ctx.save_for_backward(x, y if relu else None, weight, mean, invstd)
        ctx.mark_non_differentiable(mean, invstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        if not ctx.training:
            raise RuntimeError("batch_norm_act: backward through evaluation-mode statistics is not supported; "
                               "use torch.nn.functional.batch_norm")
        x, y, weight, mean, invstd = ctx.saved_tensors
        dx, dw, db, dres = torch.ops.blackwell.batch_norm_act_backward(dy, x, y, weight, mean, invstd, ctx.relu,
                                                                       ctx.has_res)
        return (dx, dw if weight is not None else None, db if weight is not None else None, None, None,
                dres if ctx.has_res else None, None, None, None, None)


def _bn_act_fast(x, weight, bias, running_mean, running_var) -> bool:
    if not _on_device(x) or x.dtype not in (torch.bfloat16, torch.float16):
        return False
    if x.dim() == 4:
        if not x.is_contiguous(memory_format=torch.channels_last):
            return False
    elif x.dim() != 2 or not x.is_contiguous():
        return False
    if x.shape[1] % 8 != 0:
        return False
    return all(t is None or t.dtype == torch.float32 for t in (weight, bias, running_mean, running_var))


def batch_norm_act(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                   running_mean: Optional[torch.Tensor], running_var: Optional[torch.Tensor],
                   residual: Optional[torch.Tensor] = None, training: bool = True, momentum: float = 0.1,
                   eps: float = 1e-5, relu: bool = True) -> torch.Tensor:
    """``act(batch_norm(x) + residual)`` with ``act`` = ReLU or identity.

    On the device, for bf16/fp16 channels-last activations with fp32 parameters, the whole expression is one
    statistics pass plus one fused normalise/affine/add/ReLU pass (and the mirrored two passes backward);
    anywhere else it is the plain composition."""
    if _bn_act_fast(x, weight, bias, running_mean, running_var) and (residual is None or (
            residual.dtype == x.dtype and residual.shape == x.shape and residual.stride() == x.stride())):
        if training or (running_mean is not None and running_var is not None and not torch.is_grad_enabled()):
            return _BatchNormAct.apply(x, weight, bias, running_mean, running_var, residual, training, momentum, eps,
                                       relu)
    y = F.batch_norm(x, running_mean, running_var, weight, bias, training, momentum, eps)
    if residual is not None:
        y = y + residual
    return F.relu(y) if relu else y


# ------------------------------------------------------------------------- RoPE
def precompute_rope_cache(seq_len: int, head_dim: int, theta: float = 10000.0, device=None):
    """fp32 ``cos``/``sin`` tables of shape [seq_len, head_dim // 2]."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device="cpu") / head_dim))
    t = torch.arange(seq_len, dtype=torch.float32, device="cpu")
    freqs = torch.outer(t, inv)
    cos, sin = freqs.cos().contiguous(), freqs.sin().contiguous()
    if device is not None:
        cos, sin = cos.to(device), sin.to(device)
    return cos, sin


def _rope_reference(x, cos, sin, positions, interleaved, conj):
    # x [B, S, H, D]; cos/sin [P, D/2]
    B, S, H, D = x.shape
    if positions is not None:
        c = cos[positions.reshape(B, S)].unsqueeze(2)
        s = sin[positions.reshape(B, S)].unsqueeze(2)
    else:
        c = cos[:S].view(1, S, 1, D // 2)
        s = sin[:S].view(1, S, 1, D // 2)
    if conj:
        s = -s
    xf = x.float()
    if interleaved:
        x0, x1 = xf[..., 0::2], xf[..., 1::2]
        o0, o1 = x0 * c - x1 * s, x1 * c + x0 * s
        out = torch.stack((o0, o1), dim=-1).flatten(-2)
    else:
        x0, x1 = xf[..., : D // 2], xf[..., D // 2:]
        out = torch.cat((x0 * c - x1 * s, x1 * c + x0 * s), dim=-1)
    return out.to(x.dtype)


def _rope_rotate_half(x, cos, sin, positions):
    """The usual library formulation (four elementwise kernels, in the input dtype): ``x * cos + rotate_half(x) * sin``
    with full-width tables.  What a stock CUDA run of this model uses."""
    B, S, H, D = x.shape
    if positions is not None:
        c, s = cos[positions.reshape(B, S)].unsqueeze(2), sin[positions.reshape(B, S)].unsqueeze(2)
    else:
        c, s = cos[:S].view(1, S, 1, D // 2), sin[:S].view(1, S, 1, D // 2)
    c = torch.cat((c, c), dim=-1).to(x.dtype)
    s = torch.cat((s, s), dim=-1).to(x.dtype)
    x0, x1 = x[..., : D // 2], x[..., D // 2:]
    return x * c + torch.cat((-x1, x0), dim=-1) * s


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin, positions, interleaved):
        ctx.save_for_backward(cos, sin, positions if positions is not None else torch.empty(0))
        ctx.has_pos = positions is not None
        ctx.interleaved = interleaved
        return torch.ops.blackwell.rope(x, cos, sin, positions, interleaved, False)

    @staticmethod
    def backward(ctx, dy):
        cos, sin, pos = ctx.saved_tensors
        dx = torch.ops.blackwell.rope(dy, cos, sin, pos if ctx.has_pos else None, ctx.interleaved, True)
        return dx, None, None, None, None


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None,
         interleaved: bool = False) -> torch.Tensor:
    """Rotary position embedding of ``x`` [batch, seq, heads, head_dim].

    ``interleaved=False`` rotates the two halves of the head dimension (Llama / NeoX layout),
    ``True`` rotates adjacent pairs (GPT-J layout). Backward is the conjugate rotation."""
    if _on_device(x):
        return _Rope.apply(x, cos, sin, positions, interleaved)
    if x.is_cuda and not interleaved and x.dtype in (torch.bfloat16, torch.float16):
        return _rope_rotate_half(x, cos, sin, positions)
    return _rope_reference(x, cos, sin, positions, interleaved, False)


# ------------------------------------------------------------------------- SwiGLU
class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return torch.ops.blackwell.swiglu(x)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        return torch.ops.blackwell.swiglu_backward(dy, x)


class _SwiGLURows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, counts):
        ctx.save_for_backward(x, counts)
        return torch.ops.blackwell.swiglu_rows(x, counts)

    @staticmethod
    def backward(ctx, dy):
        x, counts = ctx.saved_tensors
        return torch.ops.blackwell.swiglu_rows_backward(dy, x, counts), None


def swiglu(x: torch.Tensor, row_counts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``silu(x[..., :h]) * x[..., h:]`` for a packed gate|up tensor.  ``row_counts`` (int32, on the device): the
    lengths of the packed row groups of a 2-D ``x``; only the first ``row_counts.sum()`` rows are computed (and get a
    gradient), the others are left as they are -- the sum is taken on the device."""
    if _on_device(x):
        if row_counts is not None:
            return _SwiGLURows.apply(x, row_counts.to(torch.int32))
        return _SwiGLU.apply(x)
    g, u = x.chunk(2, dim=-1)
    return F.silu(g) * u


gated_silu = swiglu


# ------------------------------------------------------------------------- grouped linear (expert GEMMs)
def _grouped_rows(counts: torch.Tensor, rows: int):
    out, start = [], 0
    for n in counts.tolist():
        n = max(0, min(int(n), rows - start))
        out.append((start, n))
        start += n
    return out


class _GroupedLinear(torch.autograd.Function):
    """``y[r] = x[r] @ w[g(r)].T`` over packed row groups whose lengths (``counts``, int32) stay on the device: one
    grouped tensor-core GEMM each for the product, the input gradient and the per-group weight gradients."""

    @staticmethod
    def forward(ctx, x, w, counts, out, grad_input_out):
        ctx.save_for_backward(x, w, counts)
        ctx.grad_input_out = grad_input_out
        if out is not None:
            ctx.mark_dirty(out)
            return torch.ops.blackwell.grouped_mm_out(x, w, counts, 0, out)
        return torch.ops.blackwell.grouped_mm(x, w, counts, 0)

    @staticmethod
    def backward(ctx, dy):
        x, w, counts = ctx.saved_tensors
        dy = dy.contiguous()
        dx = None
        if ctx.needs_input_grad[0]:
            if ctx.grad_input_out is not None:
                dx = torch.ops.blackwell.grouped_mm_out(dy, w, counts, 1, ctx.grad_input_out)
            else:
                dx = torch.ops.blackwell.grouped_mm(dy, w, counts, 1)
        dw = torch.ops.blackwell.grouped_mm(dy, x, counts, 2) if ctx.needs_input_grad[1] else None
        return dx, dw, None, None, None


def grouped_linear(x: torch.Tensor, w: torch.Tensor, counts: torch.Tensor, out: Optional[torch.Tensor] = None,
                   grad_input_out: Optional[torch.Tensor] = None):
    """Rows of ``x`` [R, K] are packed group after group (``counts[g]`` rows for group g); ``w`` is [G, N, K].
    Returns [R, N]; rows past ``counts.sum()`` are left as they are (uninitialised without ``out``).  On the
    blackwell device nothing reads ``counts`` on the host.  ``out`` / ``grad_input_out`` name buffers the product /
    the input gradient are written into (an exchange arena, so that no copy follows)."""
    if _on_device(x) and x.dtype in (torch.bfloat16, torch.float16):
        return _GroupedLinear.apply(x, w, counts.to(torch.int32), out, grad_input_out)
    parts = [F.linear(x[s:s + n], w[g]) for g, (s, n) in enumerate(_grouped_rows(counts, x.shape[0]))]
    used = sum(p.shape[0] for p in parts)
    y = torch.cat(parts + [x.new_zeros((x.shape[0] - used, w.shape[1]))], 0)
    if out is not None:
        out.copy_(y)
        return out
    return y


class _SiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        return torch.ops.blackwell.silu_mul(gate, up)

    @staticmethod
    def backward(ctx, dy):
        gate, up = ctx.saved_tensors
        return torch.ops.blackwell.silu_mul_backward(dy, gate, up)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` in one kernel (two-tensor SwiGLU)."""
    if _on_device(gate):
        return _SiluMul.apply(gate, up)
    return F.silu(gate) * up


# ------------------------------------------------------------------------- cross entropy
def _mean_of_counted(loss_rows, target, ignore_index):
    """(mean over the rows that count, their number), in one launch.  Row shards are added up where they are instead: the
    one-launch operation would have to gather losses and targets first."""
    if DTensor is not None and isinstance(loss_rows, DTensor):
        n = (target != ignore_index).sum().clamp_min(1).to(torch.float32)
        return loss_rows.sum() / n, n
    return torch.ops.blackwell.cross_entropy_mean(loss_rows, target, ignore_index)


class _FusedCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index, label_smoothing, reduction, inplace_backward):
        loss_rows, lse = torch.ops.blackwell.cross_entropy_fwd(logits, target, ignore_index, label_smoothing)
        n_valid = None
        if reduction == "mean":
            out, n_valid = _mean_of_counted(loss_rows, target, ignore_index)
        elif reduction == "sum":
            out = loss_rows.sum()
        else:
            out = loss_rows
        ctx.save_for_backward(logits, lse, target, n_valid if n_valid is not None else torch.empty(0))
        ctx.cfg = (ignore_index, label_smoothing, reduction, inplace_backward)
        return out

    @staticmethod
    def backward(ctx, dloss):
        logits, lse, target, n_valid = ctx.saved_tensors
        ignore_index, ls, reduction, inplace = ctx.cfg
        g = dloss.to(torch.float32)
        if reduction == "mean":
            g = g / n_valid
        g = g.reshape(-1) if reduction == "none" else g.reshape(1)
        if inplace and logits.is_contiguous():
            dl = torch.ops.blackwell.cross_entropy_bwd_(logits, lse, target, g, 1.0, ignore_index, ls)
        else:
            dl = torch.ops.blackwell.cross_entropy_bwd(logits, lse, target, g, 1.0, ignore_index, ls)
        return dl, None, None, None, None, None


def fused_cross_entropy(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                        label_smoothing: float = 0.0, reduction: str = "mean",
                        inplace_backward: bool = False) -> torch.Tensor:
    """Cross entropy over [T, V] logits that never materialises the probabilities.

    Forward stores only the per-row log-sum-exp; backward regenerates softmax from it.
    ``inplace_backward=True`` writes the gradient over the logits (saves T*V elements) --
    only valid when nothing else needs the logits after the loss."""
    if logits.dim() != 2:
        logits = logits.reshape(-1, logits.shape[-1])
        target = target.reshape(-1)
    if _on_device(logits):
        return _FusedCE.apply(logits, target, ignore_index, label_smoothing, reduction, inplace_backward)
    return F.cross_entropy(logits.float(), target, ignore_index=ignore_index, label_smoothing=label_smoothing,
                           reduction=reduction)


# ------------------------------------------------------------------------- misc
def multi_tensor_l2norm(tensors: List[torch.Tensor], per_tensor: bool = False):
    """Global (and optionally per-tensor) L2 norm of a list of tensors in a few launches."""
    if len(tensors) > 0 and _on_device(tensors[0]):
        total, per = torch.ops.blackwell.multi_tensor_l2norm(list(tensors), per_tensor)
        return (total, per) if per_tensor else (total, None)
    per = torch.stack([t.float().norm(2) for t in tensors]) if tensors else torch.zeros(0)
    return per.norm(2).reshape(1), (per if per_tensor else None)


def scaled_dot_product_attention(q, k, v, attn_mask=None, dropout_p: float = 0.0, is_causal: bool = False,
                                 scale: Optional[float] = None, enable_gqa: bool = False):
    """``F.scaled_dot_product_attention``; on the device it is routed to the backend's attention kernels."""
    return F.scaled_dot_product_attention(q, k, v, attn_mask=attn_mask, dropout_p=dropout_p, is_causal=is_causal,
                                          scale=scale, enable_gqa=enable_gqa)


# ------------------------------------------------------------------------- windowed and packed variable-length attention
def _check_window(causal: bool, window: Optional[int], sinks: int, scale: Optional[float]) -> None:
    if scale is not None and window is not None and not 0 < scale < math.inf:
        raise ValueError(f"the softmax scale must be positive, got {scale}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    if window is not None:
        if window <= 0:
            raise ValueError(f"window must be positive, got {window}")
        if not causal:
            raise ValueError("a window needs causal=True")


def _window_mask(sq: int, sk: int, window: Optional[int], sinks: int, device) -> torch.Tensor:
    """[sq, sk], true where query i sees key j: ``j <= i and (i - j < window or j < sinks)``."""
    i, j = torch.arange(sq, device=device)[:, None], torch.arange(sk, device=device)[None, :]
    seen = j <= i
    return seen if window is None else seen & ((i - j < window) | (j < sinks))


def _native_attention(q, k, v) -> bool:
    return (_on_device(q) and q.shape[-1] == 128 and q.dtype in (torch.bfloat16, torch.float16)
            and k.dtype == q.dtype and v.dtype == q.dtype)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale):
        out, lse, rest = torch.ops.blackwell.window_attention_with_remainder(q, k, v, window, sinks, scale)
        ctx.save_for_backward(q, k, v, out, lse, rest)
        ctx.args = (window, sinks, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        *saved, rest = ctx.saved_tensors
        dq, dk, dv = torch.ops.blackwell.window_attention_backward(d_out, *saved, *ctx.args, rest)
        return dq, dk, dv, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention with a sliding window and a few first tokens that stay visible: query i sees key j when
    ``j <= i and (i - j < window or j < sinks)``.  ``q`` [B, Sq, H, D], ``k`` / ``v`` [B, Sk, Hkv, D] (Hkv divides H);
    returns [B, Sq, H, D], zeros for a query that sees no key.  On the blackwell device with D = 128 and bf16 / fp16 the
    tensor-core kernels skip the blocks of keys outside the mask, in both directions; otherwise it is
    ``scaled_dot_product_attention`` with the mask.  There the gradient of ``q`` is summed in 32 bits in the order in which
    blocks of keys arrive, which ``torch.use_deterministic_algorithms`` refuses, and what is not finite reaches further than the mask:
    queries and keys are taken in blocks of 128 from the start of a sequence, and where any query of a block sees any key of another,
    an infinity or NaN in a value of the one reaches the outputs and gradients of all queries of the other, one in a key the
    gradients of all of them, one in a query or an incoming gradient those of all keys.  Other blocks, heads, sequences and batches
    are not reached.  A call that is to be differentiated keeps a second tensor like the output: what rounding left of it."""
    _check_window(True, window, sinks, softmax_scale)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"window_attention: q [B, Sq, H, D] and k, v [B, Sk, Hkv, D] with Hkv a divisor of H expected, got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if _native_attention(q, k, v):
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _WindowAttention.apply(q, k, v, int(window), int(sinks), softmax_scale)
        return torch.ops.blackwell.window_attention(q, k, v, int(window), int(sinks), softmax_scale)[0]
    rep = q.shape[2] // k.shape[2]
    kt, vt = k.transpose(1, 2), v.transpose(1, 2)
    if rep > 1:
        kt, vt = kt.repeat_interleave(rep, 1), vt.repeat_interleave(rep, 1)
    mask = _window_mask(q.shape[1], k.shape[1], window, sinks, q.device)
    return F.scaled_dot_product_attention(q.transpose(1, 2), kt, vt, attn_mask=mask, scale=softmax_scale).transpose(1, 2)


class _VarlenAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, window, sinks):
        rest = None
        if window is not None and any(ctx.needs_input_grad):
            out, lse, rest = torch.ops.blackwell.varlen_attention_with_remainder(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, scale)
        else:
            out, lse = torch.ops.blackwell.varlen_attention(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, window, sinks)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k, rest)
        ctx.args = (max_q, max_k, causal, scale, window, sinks)
        return out

    @staticmethod
    def backward(ctx, d_out):
        q, k, v, out, lse, cu_q, cu_k, rest = ctx.saved_tensors
        dq, dk, dv = torch.ops.blackwell.varlen_attention_backward(d_out, q, k, v, out, lse, cu_q, cu_k, *ctx.args, rest)
        return dq, dk, dv, None, None, None, None, None, None, None, None


class _VarlenWindowAttention(_VarlenAttention):
    backward = staticmethod(torch.autograd.function.once_differentiable(_VarlenAttention.backward))


def flash_attn_varlen_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                           cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                           softmax_scale: Optional[float] = None, causal: bool = False,
                           window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """Attention over sequences of different lengths packed without padding: ``q`` [total_q, H, D], ``k`` / ``v``
    [total_k, Hkv, D]; sequence i owns rows ``cu_seqlens[i]:cu_seqlens[i + 1]`` (int32 prefix sums, on the device of
    the tensors).  Returns [total_q, H, D].  On the blackwell device with D = 128 and bf16 / fp16 the whole batch is
    one launch of the tensor-core forward (one more for the backward) and the lengths are never read on the host;
    otherwise the sequences are processed one by one with ``scaled_dot_product_attention``.  A causal mask compares
    positions inside a sequence (key index <= query index); ``window`` and ``sinks`` narrow it as in
    ``window_attention``, and rows past the last sequence then get zeros, in the gradients too."""
    _check_window(causal, window, sinks, softmax_scale)
    if _native_attention(q, k, v):
        attention = _VarlenAttention if window is None else _VarlenWindowAttention
        return attention.apply(q, k, v, cu_seqlens_q.to(torch.int32), cu_seqlens_k.to(torch.int32),
                               int(max_seqlen_q), int(max_seqlen_k), bool(causal), softmax_scale, window, int(sinks))
    cq, ck = cu_seqlens_q.tolist(), cu_seqlens_k.tolist()
    rep = q.shape[1] // k.shape[1]
    outs = []
    for i in range(len(cq) - 1):
        qi = q[cq[i]:cq[i + 1]].transpose(0, 1).unsqueeze(0)
        ki = k[ck[i]:ck[i + 1]].transpose(0, 1).unsqueeze(0)
        vi = v[ck[i]:ck[i + 1]].transpose(0, 1).unsqueeze(0)
        if rep > 1:
            ki, vi = ki.repeat_interleave(rep, 1), vi.repeat_interleave(rep, 1)
        mask = _window_mask(qi.shape[2], ki.shape[2], window, sinks, q.device) if causal else None
        o = F.scaled_dot_product_attention(qi, ki, vi, attn_mask=mask, scale=softmax_scale)
        outs.append(o.squeeze(0).transpose(0, 1))
    if window is not None and cq[-1] < q.shape[0]:
        outs.append(q.new_zeros((q.shape[0] - cq[-1],) + tuple(q.shape[1:])))
    return torch.cat(outs, 0)


# ------------------------------------------------------------------------- paged key-value cache
def _no_grad_inputs(op: str, *tensors) -> None:      # on the device the operators say so themselves
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{op} has no gradient: call it under torch.no_grad()")


def _paged_native(q: torch.Tensor) -> bool:
    return _on_device(q) and q.dtype in (torch.bfloat16, torch.float16) and q.shape[-1] in (64, 128)


def paged_rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                     k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding (rotate-half layout) of new tokens and their paged cache update, one launch on the device.

    ``q`` [T, H, D], ``k`` / ``v`` [T, Hkv, D] hold the new tokens sequence after sequence: the same number for each, or
    ``cu_seqlens`` (int32 [B + 1]).  ``k_pages`` / ``v_pages`` [pages, Hkv, page size, D] are written in place;
    ``block_table`` (int32 [B, W]) names each sequence's pages in order; ``seq_lens`` (int32 [B]) counts the tokens in the
    cache, the new ones included: token i of n stands at position ``len - n + i``.  ``cos`` / ``sin`` are float32
    [positions, D / 2].  Returns the rotated queries.  Tokens past the last sequence or before position 0 are padding:
    zeros come back for them and nothing is written.  A page number outside the pool or a position outside the tables is
    reported by the next ``synchronize()`` (the row is not written; the last angle is used).  Sequences do not
    share the pages that they write, and the pools are not expanded tensors."""
    if _paged_native(q):
        return torch.ops.blackwell.paged_rope_cache(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, cu_seqlens)
    _no_grad_inputs("paged_rope_cache", q, k, v)
    if any(n > 1 and stride == 0 for pool in (k_pages, v_pages) for n, stride in zip(pool.shape, pool.stride())):
        raise RuntimeError("paged_rope_cache: an expanded pool cannot be written, more than one element refers to a single memory location")
    T, B, page = q.shape[0], seq_lens.shape[0], k_pages.shape[2]
    t = torch.arange(T, device=q.device)
    if cu_seqlens is None:
        n = T // max(B, 1)
        if n * B != T:
            raise RuntimeError(f"paged_rope_cache: {T} tokens do not divide over {B} sequences")
        cu = torch.arange(B + 1, device=q.device) * n
    else:
        cu = cu_seqlens.long()
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, max(B - 1, 0))
    if B == 0:
        return torch.zeros_like(q)
    from_end = cu[seq + 1] - t
    pos = seq_lens.long()[seq] - from_end
    real = (from_end > 0) & (t >= cu[seq]) & (pos >= 0)
    index = torch.div(pos.clamp_min(0), page, rounding_mode="floor")
    inside = index < block_table.shape[1]
    number = torch.full_like(index, -1) if block_table.shape[1] == 0 else torch.where(
        inside, block_table.long()[seq, index.clamp_max(block_table.shape[1] - 1)], -1)
    bad = real & ((number < 0) | (number >= k_pages.shape[0]))
    late = real & (pos >= cos.shape[0])
    if not _on_device(q) and bool((bad | late).any()):
        raise IndexError("paged_rope_cache: a token's page or position does not exist")
    angle = pos.clamp(0, cos.shape[0] - 1)
    c, s, half = cos[angle][:, None], sin[angle][:, None], q.shape[-1] // 2

    def rotate(x):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat((a * c - b * s, b * c + a * s), -1).to(x.dtype)

    keep = real & ~bad
    rows = (number[keep], slice(None), (pos % page)[keep])
    k_pages[rows] = rotate(k)[keep]
    v_pages[rows] = v[keep]
    return rotate(q).masked_fill(~real[:, None, None], 0)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                    softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the n newest tokens of each sequence (``q`` [B, n, H, D]; n = 1 when decoding, more when drafted tokens
    are checked) over a paged cache as ``paged_rope_cache`` writes it.  Token i sees the keys up to its own position
    ``len - n + i``; ``window`` / ``sinks`` narrow that as in ``window_attention``.  Only pages with a visible key are
    read: others may already belong to someone else, and their table entries may be anything.  A token that sees no key
    (an empty sequence) gets zeros.  The keys of a page number outside the pool are hidden, which the next ``synchronize()``
    reports."""
    _check_window(True, window, sinks, softmax_scale)
    if softmax_scale is not None and not 0 < softmax_scale < math.inf:
        raise ValueError(f"the softmax scale must be positive, got {softmax_scale}")
    if _paged_native(q):
        return torch.ops.blackwell.paged_attention(q, k_pages, v_pages, block_table, seq_lens, window, sinks, softmax_scale)
    _no_grad_inputs("paged_attention", q, k_pages, v_pages)
    B, n, H, D = q.shape
    pages, Hkv, page, _ = k_pages.shape
    L = block_table.shape[1] * page
    if L == 0 or q.numel() == 0:
        return torch.zeros_like(q)
    table = block_table.long()
    j = torch.arange(L, device=q.device)
    pos = (seq_lens.long().clamp(0, L)[:, None] - n + torch.arange(n, device=q.device))[:, :, None]
    seen = j <= pos
    if window is not None:
        seen = seen & ((pos - j < window) | (j < sinks))
    there = ((table >= 0) & (table < pages)).repeat_interleave(page, 1)[:, None]
    if not _on_device(q) and bool((seen & ~there).any()):
        raise IndexError("paged_attention: a visible key's page does not exist")
    seen = (seen & there)[:, None, None]                                                        # [B, 1, 1, n, L]
    some = seen.any(3, keepdim=True).squeeze(3)[..., None]                                      # keys that any token sees
    index = table.clamp(0, max(pages - 1, 0))

    def rows(pool):
        x = pool[index] if pages else pool.new_zeros((B, table.shape[1], Hkv, page, D))
        return x.transpose(1, 2).reshape(B, Hkv, 1, L, D).float().masked_fill(~some, 0)

    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    x = (q.float().view(B, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4) @ rows(k_pages).transpose(-1, -2)) * scale
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top.masked_fill(top == float("-inf"), 0))
    v = rows(v_pages)
    odd = ~torch.isfinite(v)
    if n == 1 or (not _on_device(q) and not bool(odd.any())):
        out = x @ v
    else:            # an infinity or NaN reaches the tokens that see it and no others: zero times it would be NaN
        weight = (x > 0).float()
        high, low, nan = (weight @ t.float() > 0 for t in (v == math.inf, v == -math.inf, v != v))
        out = (x @ v.masked_fill(odd, 0)).masked_fill(high, math.inf).masked_fill(low, -math.inf).masked_fill(nan | (high & low), math.nan)
    out = out / x.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(q.dtype)


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                  draft_probs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Checks drafted tokens against the target model's probabilities with given random numbers, so that what comes out is
    distributed as if it were sampled from the target alone.

    ``target_probs`` [B, n + 1, V] (the rows for the n drafted tokens and the one after them), ``draft_tokens`` int64 [B, n],
    ``uniforms`` float32 [B, n + 1] in [0, 1), ``draft_probs`` [B, n, V] in the type of ``target_probs`` or None for drafts that
    were certain (a greedy draft).  Draft i is taken while ``uniforms[i] * draft_probs[i, x_i] < target_probs[i, x_i]``;
    at the first refusal r one token is drawn from ``max(target_probs[r] - draft_probs[r], 0)``, after n taken drafts from
    ``target_probs[n]``: the first token at which the running sum exceeds ``uniforms[n]`` times the whole (a number below
    zero or NaN counts as zero there, from one on it is the last token that has weight).  A draft outside the vocabulary
    (-1, say) ends a sequence's draft early: the token there is drawn from the target's row.  Sums are held in 64 bits.

    Returns ``(taken [B], tokens [B, n + 1])``, both int64: the taken drafts, the drawn token, then -1.  Where a row has no
    weight at all (zeros or NaN) the drawn token is -1."""
    if _on_device(target_probs) and target_probs.dtype in (torch.float32, torch.bfloat16, torch.float16):
        return torch.ops.blackwell.verify_drafts(target_probs, draft_tokens, uniforms, draft_probs)
    _no_grad_inputs("verify_drafts", target_probs, draft_probs)
    B, n1, V = target_probs.shape
    n, x, u = n1 - 1, draft_tokens, uniforms.double()
    if tuple(x.shape) != (B, n) or tuple(u.shape) != (B, n1) or (draft_probs is not None and tuple(draft_probs.shape) != (B, n, V)):
        raise RuntimeError("verify_drafts: draft_tokens [B, n], uniforms [B, n + 1] and draft_probs [B, n, V] expected")
    if x.dtype != torch.long or uniforms.dtype != torch.float32 or (draft_probs is not None and draft_probs.dtype != target_probs.dtype):
        raise RuntimeError("verify_drafts: draft_tokens must be int64, uniforms float32 and draft_probs of target_probs' type")
    known = (x >= 0) & (x < V)
    at = x.clamp(0, V - 1)[..., None]
    p = target_probs[:, :n].gather(2, at).squeeze(2).double()
    q = draft_probs.gather(2, at).squeeze(2).double() if draft_probs is not None else torch.ones_like(p)
    taken = (known & (u[:, :n] * q < p)).long().cumprod(1).sum(1)
    row = torch.arange(B, device=x.device)
    w = target_probs[row, taken].double()
    if n > 0:
        stop = taken.clamp_max(n - 1)
        less = w - draft_probs[row, stop].double() if draft_probs is not None else w.scatter(1, at[row, stop], 0.0)
        less = torch.where(less > 0, less, 0.0)
        refused = (taken < n) & known[row, stop] & (less.sum(1) > 0)
        w = torch.where(refused[:, None], less, w)
    w = torch.where(w > 0, w, 0.0)
    total = w.cumsum(1)
    past = (w > 0) & (total > torch.where(u[:, n:] > 0, u[:, n:], 0.0) * total[:, -1:])
    last = ((w > 0) * torch.arange(V, device=x.device)).amax(1)
    token = torch.where(past.any(1), past.long().argmax(1), last)
    token = torch.where(total[:, -1] > 0, token, -1)
    i = torch.arange(n1, device=x.device)
    drafts = torch.cat((x, x.new_full((B, 1), -1)), 1)
    return taken, torch.where(i < taken[:, None], drafts, torch.where(i == taken[:, None], token[:, None], -1))
