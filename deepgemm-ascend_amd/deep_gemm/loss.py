"""Cross entropy of a linear layer over a large vocabulary, without keeping the logits.

    loss, lse = linear_cross_entropy(x, weight, target)
    d_x, d_weight = linear_cross_entropy_backward(d_loss, x, weight, target, lse)

No autograd graph is recorded: the results of inputs that require gradients have none, and a program makes the second call itself.
The forward pass holds a maximum and a sum for each token and tile of words; the backward pass computes the logits again, a
piece of the vocabulary at a time, and holds the gradient of one piece in bf16.
"""
import ctypes
from typing import Tuple

import torch

from . import _lib
from .gemm import _operators, _stream
from .layout import _assert
from .runtime import cu_cap, get_dry_run

MAX_TOKENS = 1 << 20


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous, 16-byte aligned rows."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.size(1) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _args(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int):
    """(GEMM-ready x, weight and target; dg_linear_xent_args over them)"""
    _assert(x.dim() == 2 and weight.dim() == 2 and x.is_cuda, 'x [T, H] and weight [V, H] must be device tensors')
    _assert(x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16, 'x and weight must be bf16')
    _assert(x.size(1) == weight.size(1), f"Conflicting shape dimension 'h': x gives {x.size(1)}, weight gives {weight.size(1)}")
    _assert(x.size(1) > 0 and x.size(1) % 8 == 0, f'H must be a multiple of 8, got {x.size(1)}')
    _assert(0 < weight.size(0) <= 2 ** 30, 'the vocabulary must have between 1 and 2^30 words')
    _assert(x.size(0) <= MAX_TOKENS, f'at most {MAX_TOKENS} tokens')
    _assert(target.dtype in (torch.int32, torch.int64) and target.shape == x.shape[:1], 'target must be a [T] int32 or int64 tensor')
    _assert(weight.device == x.device and target.device == x.device, 'x, weight and target must be on the same device')
    x, weight, target = _rows(x), _rows(weight), target.contiguous()
    a = _lib.LinearXentArgs()
    a.tokens, a.width, a.vocab = x.size(0), x.size(1), weight.size(0)
    a.x, a.x_ld, a.w, a.w_ld = x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0)
    a.target, a.target_bytes, a.ignore_index = target.data_ptr(), target.element_size(), ignore_index
    a.num_cus = cu_cap()
    return (x, weight, target), a


def _run(fn: str, a: _lib.LinearXentArgs, backward: int, x: torch.Tensor) -> None:
    _lib.raise_pending()
    lib = _lib.load()
    need = ctypes.c_int64()
    _lib.check(lib.dg_linear_xent_workspace_size(a, backward, ctypes.byref(need)), lib)
    ws = torch.empty(need.value, dtype=torch.uint8, device=x.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    _lib.check(getattr(lib, fn)(a, _stream(x)), lib)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [T], lse [T]) in fp32 of the logits ``x @ weight^T`` (x [T, H], weight [V, H] bf16, H a multiple of 8): the log of
    the sum of a token's exponentials, and that minus the target's logit.

    A token whose target is ``ignore_index`` has loss 0; a target outside the vocabulary counts as ignored and is reported
    (``check_errors``)."""
    ext = _operators(x)
    if ext is not None:
        made = ext.linear_xent(x, weight, target, ignore_index, cu_cap(), _stream(x))
        if made:
            return made[0], made[1]
    keep, a = _args(x, weight, target, ignore_index)
    loss, lse = (torch.empty(x.size(0), dtype=torch.float32, device=x.device) for _ in range(2))
    if x.size(0) == 0 or get_dry_run():
        return loss, lse
    a.loss, a.lse = loss.data_ptr(), lse.data_ptr()
    _run('dg_linear_xent_forward', a, 0, x)
    return loss, lse


def linear_cross_entropy_backward(d_loss: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                                  lse: torch.Tensor, ignore_index: int = -100) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients (d_x [T, H], d_weight [V, H]) in bf16 of the losses weighted by ``d_loss`` [T] fp32 (1 / T for a mean over T
    tokens), with ``lse`` as ``linear_cross_entropy`` gave it.

    The gradient of the logits is rounded to bf16 for both products; the target's entries of it count in full in d_x, and in d_weight
    where the weights are equal (relative errors 0.0017, and 0.0022 in d_weight with weights drawn from (0, 1))."""
    ext = _operators(x)
    if ext is not None:
        made = ext.linear_xent_backward(d_loss, x, weight, target, lse, ignore_index, cu_cap(), _stream(x))
        if made:
            return made[0], made[1]
    keep, a = _args(x, weight, target, ignore_index)
    for name, t in (('d_loss', d_loss), ('lse', lse)):
        _assert(t.dtype == torch.float32 and t.shape == x.shape[:1] and t.device == x.device, f'{name} must be a [T] fp32 tensor')
    d_x = torch.empty((x.size(0), x.size(1)), dtype=torch.bfloat16, device=x.device)
    if x.size(0) == 0:
        return d_x, torch.zeros((weight.size(0), weight.size(1)), dtype=torch.bfloat16, device=x.device)
    d_w = torch.empty((weight.size(0), weight.size(1)), dtype=torch.bfloat16, device=x.device)
    if get_dry_run():
        return d_x, d_w
    d_loss, lse = d_loss.contiguous(), lse.contiguous()
    a.lse, a.d_loss = lse.data_ptr(), d_loss.data_ptr()
    a.d_x, a.d_w, a.d_x_ld, a.d_w_ld = d_x.data_ptr(), d_w.data_ptr(), d_x.size(1), d_w.size(1)
    _run('dg_linear_xent_backward', a, 1, x)
    return d_x, d_w
