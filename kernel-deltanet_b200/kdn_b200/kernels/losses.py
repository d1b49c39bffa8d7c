"""Losses over vocabulary logits on libkdn, forward and backward (CUDA tensors only).

What follows upcycling: distilling the teacher into the student, then preference or policy tuning, and the
token log-probabilities that those need of a reference or a sampling policy.  With x = logits / temperature and
q = softmax(x):

* ``token_logprobs(logits, labels)`` -> log q[label] of every row (differentiable).
* ``policy_loss(logits, actions, old_logps, advantages, ...)`` -> (loss, logps, entropy): the clipped policy loss,
  with a KL term to ``ref_logps`` and an entropy bonus.
* ``preference_loss(logits, labels, cu_seqlens, ref_logps, ...)`` -> (loss, log_ratios, logps): the logistic loss of
  paired log ratios over packed sequences 2 p (preferred) and 2 p + 1.
* ``distillation_loss(logits, teacher_logits, teacher_ids, ...)`` -> (loss, divergence): KL divergence from a teacher
  of which the largest logits of each row are known.

Logits are float32 or bfloat16, [..., vocab], with any row stride and alignment; the formulas, what ignored rows,
weights and padding mean, and what -inf and NaN give stand at the entries of include/kdn.h.  Only logits receive a
gradient, and in reverse mode alone: logits with a forward-mode tangent are refused.  The loss and its gradient come
from one pass over the logits (two for ``preference_loss``), so ``loss.backward()`` only hands over what the forward
formed (scaled by the upstream gradient where that is not one); the logits are not kept.  The gradient has the logits'
type: a factor that is no power of two rounds a bf16 one a second time (put it into ``weights``, where it costs nothing).
A second backward through one call raises.  ``*_loss_and_grad`` return the gradient directly, as a last value, for
trainers that run their own head backward.  Losses, log-probabilities and statistics are float32.  Errors raise
RuntimeError; there is no CPU path.

Logits that no view makes [n, vocab] rows are copied: ``logits[:, :-1]`` of a [B, T, vocab] tensor is.  Pass all of them,
with ignore_index as the label of the positions that predict nothing.  Logits whose first row starts off 16 bytes while
their rows lie whole 16 bytes apart (``logits[:, 1:]`` of [n, vocab]) get a gradient of another 16-byte phase, stored element by element.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as fwad
from torch.autograd.function import once_differentiable

from .. import _lib

_INDEX = {torch.int64: _lib.KDN_INDEX_I64, torch.int32: _lib.KDN_INDEX_I32}
_DTYPE = {torch.float32: _lib.KDN_DTYPE_F32, torch.bfloat16: _lib.KDN_DTYPE_BF16}
_entries: dict = {}


def _call(name: str, dev: torch.device, *args) -> None:
    """The C entry on dev's current stream.  A call of a few rows takes longer on the host than on the GPU: the entry is
    looked up once, and the stream's handle is asked for directly."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    i = dev.index
    if torch._C._cuda_getDevice() == i:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _lib.check(rc, name)


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """[..., V] -> [n, V] with unit-stride rows (a view wherever the strides allow one)."""
    if not logits.is_cuda:
        raise RuntimeError("kdn_b200 runs on CUDA tensors only (no CPU fallback)")
    if logits.dtype not in _DTYPE:
        raise RuntimeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.dim() < 2 or logits.shape[-1] < 1:
        raise RuntimeError(f"logits must be [..., vocab], got {tuple(logits.shape)}")
    if fwad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("the losses over logits have no forward-mode derivative")
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if z.stride(1) != 1 and z.shape[1] > 1 or z.shape[0] > 1 and z.stride(0) < z.shape[1]:
        z = z.contiguous()
    return z


def _ld(z: torch.Tensor) -> int:
    return z.stride(0) if z.shape[0] > 1 else z.shape[1]


def _index(t: torch.Tensor, shape, dev, name: str) -> torch.Tensor:
    if t.dtype not in _INDEX:
        raise RuntimeError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.shape != shape:
        raise RuntimeError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, logits on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _per_row(t: Optional[torch.Tensor], shape, dev, name: str) -> Optional[torch.Tensor]:
    """A float value per row, as contiguous float32."""
    if t is None:
        return None
    if t.shape != shape:
        raise RuntimeError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, logits on {dev}")
    if t.dtype != torch.float32:
        if not t.dtype.is_floating_point:
            raise RuntimeError(f"{name} must be floating point, got {t.dtype}")
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _grad_rows(z: torch.Tensor) -> torch.Tensor:
    """The gradient's buffer [n, V]: rows padded to 16 bytes where z's rows start on 16 bytes, else rows of the same
    16-byte phase as z's, so that both move by the same vectors."""
    n, V = z.shape
    per16 = 16 // z.element_size()
    ld = _ld(z)
    if ld % per16 == 0 or n <= 1:
        width = (V + per16 - 1) // per16 * per16
    else:
        width = V + (ld - V) % per16
    buf = torch.empty(n, width, device=z.device, dtype=z.dtype)
    return buf if width == V else buf[:, :V]


def _f32(shape, dev: torch.device) -> torch.Tensor:
    return torch.empty(shape, device=dev, dtype=torch.float32)


def _buffers(workspace: int, dev: torch.device, *shapes):
    """A workspace of `workspace` bytes (a multiple of 256) and float32 outputs of the given shapes.  Each is an
    allocation of its own: views of one buffer share a version counter, and writing to one of them in place would
    invalidate a graph that has kept another."""
    ws = torch.empty(workspace >> 2, device=dev, dtype=torch.float32)
    return (ws, *[ws.new_empty(s) for s in shapes])


def _scalar_grad(holder: list, dloss: torch.Tensor) -> torch.Tensor:
    """The gradient that a forward formed, scaled in place by the upstream gradient of the loss."""
    if not holder:
        raise RuntimeError("the gradient of this loss has been handed over already: call the loss again to go "
                           "backward a second time")
    g = holder.pop()
    if g.numel():
        scale = dloss.to(torch.float32)
        _call("kdn_scale_rows", g.device, g.data_ptr(), _DTYPE[g.dtype], _ld(g), g.shape[0], g.shape[1],
              scale.data_ptr())
    return g


def _wants_grad(logits: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and logits.requires_grad


# ------------------------------------------------------------------------------------- token log-probabilities
def _token_logprobs(z, y, temperature, ignore_index, keep_stats):
    n, V = z.shape
    logps = _f32(n, z.device)
    stats = _f32((n, 2), z.device) if keep_stats else None
    _call("kdn_token_logprobs", z.device, z.data_ptr(), _DTYPE[z.dtype], _ld(z), y.data_ptr(), _INDEX[y.dtype],
          ignore_index, logps.data_ptr(), _lib.ptr(stats), n, V, temperature)
    return logps, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, y, temperature, ignore_index):
        logps, stats = _token_logprobs(z, y, temperature, ignore_index, True)
        ctx.save_for_backward(z, y, stats)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogps):
        z, y, stats = ctx.saved_tensors
        return token_logprobs_backward(z, y, stats, dlogps, ctx.temperature, ctx.ignore_index), None, None, None


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0,
                   ignore_index: int = -100) -> torch.Tensor:
    """log softmax(logits / temperature)[label] of every row: logits [..., V], labels [...] -> [...] float32; 0 where
    the label is ignore_index.  Differentiable with respect to logits (kdn_token_logprobs and its backward)."""
    z = _rows(logits)
    y = _index(labels, logits.shape[:-1], logits.device, "labels")
    shape = y.shape
    if len(shape) != 1:
        y = y.reshape(-1)
    if _wants_grad(logits):
        logps = _TokenLogprobs.apply(z, y, float(temperature), int(ignore_index))
    else:
        logps = _token_logprobs(z, y, float(temperature), int(ignore_index), False)[0]
    return logps if len(shape) == 1 else logps.view(shape)


def token_logprobs_backward(logits: torch.Tensor, labels: torch.Tensor, row_stats: torch.Tensor, dlogps: torch.Tensor,
                            temperature: float = 1.0, ignore_index: int = -100) -> torch.Tensor:
    """Gradient of token_logprobs for dlogps [n] on logits [n, V], from the row statistics [n, 2] its forward keeps
    (each row's largest logit and the sum of exponentials below it; kdn_token_logprobs_backward)."""
    z = _rows(logits)
    n, V = z.shape
    y = _index(labels, (n,), z.device, "labels")
    d = _per_row(dlogps, (n,), z.device, "dlogps")
    st = _per_row(row_stats, (n, 2), z.device, "row_stats")
    g = _grad_rows(z)
    _call("kdn_token_logprobs_backward", z.device, z.data_ptr(), _DTYPE[z.dtype], _ld(z), y.data_ptr(),
          _INDEX[y.dtype], int(ignore_index), st.data_ptr(), d.data_ptr(), g.data_ptr(), _ld(g), n, V,
          float(temperature))
    return g


# --------------------------------------------------------------------------------------------------- policy loss
def _policy(z, y, old, adv, ref, w, clip_low, clip_high, kl_coef, entropy_coef, temperature, ignore_index, with_grad):
    n, V = z.shape
    dev = z.device
    size = 256 + (4 * n + 255) // 256 * 256  # kdn_policy_loss_workspace_size
    ws, loss, logps, entropy = _buffers(size, dev, (), n, n)
    g = _grad_rows(z) if with_grad else None
    _call("kdn_policy_loss", dev, z.data_ptr(), _DTYPE[z.dtype], _ld(z), y.data_ptr(), _INDEX[y.dtype], ignore_index,
          old.data_ptr(), adv.data_ptr(), _lib.ptr(ref), _lib.ptr(w), clip_low, clip_high, kl_coef, entropy_coef,
          temperature, loss.data_ptr(), logps.data_ptr(), entropy.data_ptr(), _lib.ptr(g),
          _ld(g) if with_grad else 0, n, V, ws.data_ptr(), size)
    return loss, logps, entropy, g


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, *args):
        loss, logps, entropy, g = _policy(z, *args, True)
        ctx.holder, ctx.rest = [g], (None,) * len(args)
        ctx.mark_non_differentiable(logps, entropy)
        return loss, logps, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dlogps, _dentropy):
        return (_scalar_grad(ctx.holder, dloss), *ctx.rest)


def _policy_args(logits, actions, old_logps, advantages, ref_logps, weights, clip_low, clip_high, kl_coef,
                 entropy_coef, temperature, ignore_index):
    z = _rows(logits)
    shape, dev = logits.shape[:-1], logits.device
    y = _index(actions, shape, dev, "actions")
    old = _per_row(old_logps, shape, dev, "old_logps")
    adv = _per_row(advantages, shape, dev, "advantages")
    if old is None or adv is None:
        raise RuntimeError("old_logps and advantages are required")
    ref = _per_row(ref_logps, shape, dev, "ref_logps")
    w = _per_row(weights, shape, dev, "weights")
    return z, y, old, adv, ref, w, float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef), \
        float(temperature), int(ignore_index)


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor, *,
                ref_logps: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                temperature: float = 1.0, ignore_index: int = -100
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, logps, entropy): loss = sum_t w_t (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) +
    kl_coef (e^g - 1 - g) - entropy_coef H), r = e^(logp - old_logps), g = ref_logps - logp, over logits [..., V] and
    per-token tensors [...]; weights None is the mean over the tokens whose action is not ignore_index.  logps and
    entropy [...] carry no gradient (kdn_policy_loss)."""
    args = _policy_args(logits, actions, old_logps, advantages, ref_logps, weights, clip_low, clip_high, kl_coef,
                        entropy_coef, temperature, ignore_index)
    if _wants_grad(logits):
        loss, logps, entropy = _PolicyLoss.apply(*args)
    else:
        loss, logps, entropy, _ = _policy(*args, False)
    if logits.dim() == 2:
        return loss, logps, entropy
    shape = logits.shape[:-1]
    return loss, logps.view(shape), entropy.view(shape)


def policy_loss_and_grad(logits: torch.Tensor, actions: torch.Tensor, old_logps: torch.Tensor,
                         advantages: torch.Tensor, *, ref_logps: Optional[torch.Tensor] = None,
                         weights: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: float = 0.2,
                         kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0,
                         ignore_index: int = -100
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """policy_loss and the gradient of its loss: (loss, logps, entropy, dlogits), dlogits in logits' shape and dtype."""
    args = _policy_args(logits, actions, old_logps, advantages, ref_logps, weights, clip_low, clip_high, kl_coef,
                        entropy_coef, temperature, ignore_index)
    loss, logps, entropy, g = _policy(*args, True)
    if logits.dim() == 2:
        return loss, logps, entropy, g
    shape = logits.shape[:-1]
    return loss, logps.view(shape), entropy.view(shape), g.reshape(logits.shape)


# ----------------------------------------------------------------------------------------------- preference loss
def _preference(z, y, cu, ref, beta, label_smoothing, length_normalised, temperature, ignore_index, with_grad):
    n, V = z.shape
    dev = z.device
    pairs = (cu.numel() - 1) // 2
    size = 256 + sum((b + 255) // 256 * 256 for b in (8 * n, 4 * n, 4 * pairs))  # kdn_preference_loss_workspace_size
    ws, loss, log_ratios, logps = _buffers(size, dev, (), 2 * pairs, n)
    g = _grad_rows(z) if with_grad else None
    _call("kdn_preference_loss", dev, z.data_ptr(), _DTYPE[z.dtype], _ld(z), y.data_ptr(), _INDEX[y.dtype],
          ignore_index, cu.data_ptr(), pairs, _lib.ptr(ref), beta, label_smoothing, length_normalised, temperature,
          loss.data_ptr(), log_ratios.data_ptr(), logps.data_ptr(), _lib.ptr(g), _ld(g) if with_grad else 0, n, V,
          ws.data_ptr(), size)
    return loss, log_ratios, logps, g


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, *args):
        loss, log_ratios, logps, g = _preference(z, *args, True)
        ctx.holder, ctx.rest = [g], (None,) * len(args)
        ctx.mark_non_differentiable(log_ratios, logps)
        return loss, log_ratios, logps

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dratios, _dlogps):
        return (_scalar_grad(ctx.holder, dloss), *ctx.rest)


def _preference_args(logits, labels, cu_seqlens, ref_logps, beta, label_smoothing, length_normalised, temperature,
                     ignore_index):
    z = _rows(logits)
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be [total_tokens, vocab], got {tuple(logits.shape)}")
    dev = z.device
    y = _index(labels, logits.shape[:-1], dev, "labels")
    ref = _per_row(ref_logps, logits.shape[:-1], dev, "ref_logps")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 3 or cu_seqlens.numel() % 2 == 0:
        raise RuntimeError(f"cu_seqlens must be [2 pairs + 1] with at least one pair, got {tuple(cu_seqlens.shape)}")
    cu = _index(cu_seqlens, cu_seqlens.shape, dev, "cu_seqlens").to(torch.int64)
    return z, y, cu, ref, float(beta), float(label_smoothing), int(bool(length_normalised)), float(temperature), \
        int(ignore_index)


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, cu_seqlens: torch.Tensor,
                    ref_logps: Optional[torch.Tensor] = None, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    length_normalised: bool = False, temperature: float = 1.0, ignore_index: int = -100
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss, log_ratios [2 pairs], logps [n]) over packed sequences: logits [n, V], labels [n] (ignore_index: prompt
    and padding tokens), cu_seqlens [2 pairs + 1] on the device, sequence 2 p preferred to 2 p + 1; ref_logps [n] the
    reference model's token_logprobs (None: no reference).  log_ratios[s] = sum of logp - ref_logps over the
    sequence's tokens (their mean with length_normalised); loss = mean over pairs of -log sigmoid(beta (log_ratios[2 p]
    - log_ratios[2 p + 1])), with label_smoothing's share of the swapped pair (kdn_preference_loss)."""
    args = _preference_args(logits, labels, cu_seqlens, ref_logps, beta, label_smoothing, length_normalised,
                            temperature, ignore_index)
    if _wants_grad(logits):
        return _PreferenceLoss.apply(*args)
    return _preference(*args, False)[:3]


def preference_loss_and_grad(logits: torch.Tensor, labels: torch.Tensor, cu_seqlens: torch.Tensor,
                             ref_logps: Optional[torch.Tensor] = None, *, beta: float = 0.1,
                             label_smoothing: float = 0.0, length_normalised: bool = False, temperature: float = 1.0,
                             ignore_index: int = -100
                             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """preference_loss and the gradient of its loss: (loss, log_ratios, logps, dlogits)."""
    return _preference(*_preference_args(logits, labels, cu_seqlens, ref_logps, beta, label_smoothing,
                                         length_normalised, temperature, ignore_index), True)


# --------------------------------------------------------------------------------------------- distillation loss
def _distillation(z, t, ids, lse, w, temperature, with_grad):
    n, V = z.shape
    dev = z.device
    size = 256 + (4 * n + 255) // 256 * 256  # kdn_distillation_loss_workspace_size
    ws, loss, divergence = _buffers(size, dev, (), n)
    g = _grad_rows(z) if with_grad else None
    _call("kdn_distillation_loss", dev, z.data_ptr(), _DTYPE[z.dtype], _ld(z), t.data_ptr(), _DTYPE[t.dtype],
          ids.data_ptr(), _INDEX[ids.dtype], t.shape[-1], _lib.ptr(lse), _lib.ptr(w), temperature, loss.data_ptr(),
          divergence.data_ptr(), _lib.ptr(g), _ld(g) if with_grad else 0, n, V, ws.data_ptr(), size)
    return loss, divergence, g


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, *args):
        loss, divergence, g = _distillation(z, *args, True)
        ctx.holder, ctx.rest = [g], (None,) * len(args)
        ctx.mark_non_differentiable(divergence)
        return loss, divergence

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _ddivergence):
        return (_scalar_grad(ctx.holder, dloss), *ctx.rest)


def _distillation_args(logits, teacher_logits, teacher_ids, teacher_lse, weights, temperature):
    z = _rows(logits)
    shape, dev = logits.shape[:-1], logits.device
    if teacher_logits.shape[:-1] != shape or teacher_logits.dim() != logits.dim() or teacher_logits.shape[-1] < 1:
        raise RuntimeError(f"teacher_logits must be {tuple(shape)} + [top], got {tuple(teacher_logits.shape)}")
    if teacher_logits.device != dev:
        raise RuntimeError(f"teacher_logits is on {teacher_logits.device}, logits on {dev}")
    t = teacher_logits
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"teacher_logits must be float32 or bfloat16, got {t.dtype}")
    t = t if t.is_contiguous() else t.contiguous()
    ids = _index(teacher_ids, teacher_logits.shape, dev, "teacher_ids")
    lse = _per_row(teacher_lse, shape, dev, "teacher_lse")
    w = _per_row(weights, shape, dev, "weights")
    return z, t, ids, lse, w, float(temperature)


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *,
                      teacher_lse: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                      temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, divergence [...]): KL(teacher || student) at `temperature` of every row of logits [..., V], from the
    teacher's largest logits and their ids [..., top] (at most 1024; negative ids are padding, and a row whose first
    id is negative counts for nothing); loss = temperature^2 sum_t w_t divergence_t, weights None being the mean over
    the rows that count.  teacher_lse None renormalises the teacher over the given entries; teacher_lse [...] =
    logsumexp(all of the teacher's logits / temperature) keeps their true probabilities and compares what is left of
    both as one more class (kdn_distillation_loss)."""
    args = _distillation_args(logits, teacher_logits, teacher_ids, teacher_lse, weights, temperature)
    if _wants_grad(logits):
        loss, divergence = _DistillationLoss.apply(*args)
    else:
        loss, divergence, _ = _distillation(*args, False)
    return loss, divergence.view(logits.shape[:-1])


def distillation_loss_and_grad(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, *,
                               teacher_lse: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                               temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """distillation_loss and the gradient of its loss: (loss, divergence, dlogits)."""
    loss, divergence, g = _distillation(*_distillation_args(logits, teacher_logits, teacher_ids, teacher_lse, weights,
                                                            temperature), True)
    if logits.dim() == 2:
        return loss, divergence, g
    return loss, divergence.view(logits.shape[:-1]), g.reshape(logits.shape)
