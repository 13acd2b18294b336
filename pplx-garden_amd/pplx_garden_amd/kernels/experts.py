"""The experts' feed-forward between `dispatch()` and `combine()`: products over rows sorted by expert.

Rows lie as `P2PAllToAll.dispatch` leaves them: expert e's `expert_num_tokens[e]` rows begin where the ranges of the
experts before it end, each rounded up to `expert_padding` rows (the operator's own).  Rows between the ranges are
neither read nor written.  Without `expert_num_tokens` there is one expert, which has all rows (a dense product: a
shared expert's, say).

    expert_matmul   out[i] = x[i] W[e]^T                               weight: [experts, n, k]
    expert_gated    out[i] = silu(x[i] G[e]^T) * (x[i] U[e]^T)         weight: [experts, 2n, k], gates before ups

with rows and weights in

* `float8_e4m3fn`: `expert_x_scale` [rows, ceil(k / 128)] as dispatch writes it (any strides) and `weight_scale`
  [experts, ceil(rows of W / 128), ceil(k / 128)], one per 128 x 128 block (`quantize_weight`).  `expert_matmul` writes bfloat16,
  float16 or float32, what `combine()` reads; `expert_gated` writes float8_e4m3fn and `out_scale`, quantised as dispatch quantises,
  which the next `expert_matmul` reads.
* `bfloat16` or `float16`: `out` has the same type, and there are gradients.  `matmul` and `gated` are the same
  products for autograd.  Where the weight needs a gradient, `expert_x` has to stay as it was until backward: a receive buffer that the next
  `dispatch()` writes before that makes backward raise, as an operation in place does (every call of the operator and of this module
  raises the versions of the tensors it writes; replays of a graph and calls on bare addresses do not).  The counts may
  change, backward has a copy.

Calls enqueue kernels on the current stream of the tensors' GPU, read the counts on the GPU and can be captured into a
graph.  They allocate nothing but, where the buffer has up to 512 rows, 16 MiB of the stream's own for sums in parts.
`tokens_per_expert` is how many rows the caller expects an expert to have (default: rows of the buffer per expert; 0 is
less than one): it chooses between kernels, any counts give right results.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from pplx_garden_amd.native.p2p_all_to_all import load_extension

_BLOCK = 128
_LARGEST = 448.0   # of e4m3
_SMALLEST_AMAX = 1e-4

_native = None


def _extension():
    global _native
    if _native is None:
        _native = load_extension()
    return _native


def expert_matmul(out: torch.Tensor, expert_x: torch.Tensor, weight: torch.Tensor,
                  expert_num_tokens: Optional[torch.Tensor] = None, expert_x_scale: Optional[torch.Tensor] = None,
                  weight_scale: Optional[torch.Tensor] = None, expert_padding: int = 1,
                  tokens_per_expert: Optional[int] = None) -> None:
    """out[i] = expert_x[i] weight[e]^T for expert e's rows i."""
    (_native or _extension()).expert_matmul(out, expert_x, weight, expert_num_tokens, expert_x_scale, weight_scale,
                                            expert_padding, tokens_per_expert)


def expert_gated(out: torch.Tensor, expert_x: torch.Tensor, weight: torch.Tensor,
                 expert_num_tokens: Optional[torch.Tensor] = None, expert_x_scale: Optional[torch.Tensor] = None,
                 weight_scale: Optional[torch.Tensor] = None, out_scale: Optional[torch.Tensor] = None,
                 projections: Optional[torch.Tensor] = None, expert_padding: int = 1,
                 tokens_per_expert: Optional[int] = None) -> None:
    """out[i] = silu(g) * u for expert e's rows i, [g, u] = expert_x[i] weight[e]^T, in one kernel.  `projections`
    [rows, 2n] (bfloat16, float16) receives [g, u], which `expert_gated_grad` needs."""
    (_native or _extension()).expert_gated(out, expert_x, weight, expert_num_tokens, expert_x_scale, weight_scale, out_scale,
                                           projections, expert_padding, tokens_per_expert)


def expert_matmul_grad(grad_x: Optional[torch.Tensor], grad_weight: Optional[torch.Tensor], grad_out: torch.Tensor,
                       expert_x: torch.Tensor, weight: torch.Tensor, expert_num_tokens: Optional[torch.Tensor] = None,
                       expert_padding: int = 1) -> None:
    """grad_x[i] = grad_out[i] weight[e]; grad_weight[e] = sum of grad_out[i]^T expert_x[i] over e's rows, zero where there
    are none.  Either may be None."""
    (_native or _extension()).expert_matmul_grad(grad_x, grad_weight, grad_out, expert_x, weight, expert_num_tokens,
                                                 expert_padding)


def expert_gated_grad(grad_x: Optional[torch.Tensor], grad_weight: Optional[torch.Tensor], grad_projections: torch.Tensor,
                      grad_out: torch.Tensor, projections: torch.Tensor, expert_x: torch.Tensor, weight: torch.Tensor,
                      expert_num_tokens: Optional[torch.Tensor] = None, expert_padding: int = 1) -> None:
    """The gradient of `expert_gated` from what it wrote into `projections`.  `grad_projections` [rows, 2n] receives the gradient of
    [g, u] and may be `projections` itself; it is rounded to the tensors' type, which the two products that follow take."""
    (_native or _extension()).expert_gated_grad(grad_x, grad_weight, grad_projections, grad_out, projections, expert_x, weight,
                                                expert_num_tokens, expert_padding)


@torch.no_grad()
def quantize_weight(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weights [experts, n, k] as float8_e4m3fn codes and a float scale per 128 x 128 block: once, when a model is
    loaded.  Same rule as dispatch's for rows: scale = amax / 448, amax at least 1e-4."""
    experts, n, k = weight.shape
    nb, kb = -(-n // _BLOCK), -(-k // _BLOCK)
    codes = torch.empty((experts, n, k), dtype=torch.float8_e4m3fn, device=weight.device)
    scale = torch.empty((experts, nb, kb), dtype=torch.float32, device=weight.device)
    for e in range(experts):   # an expert at a time: the float copy of all of them may not fit
        w = torch.nn.functional.pad(weight[e].float(), (0, kb * _BLOCK - k, 0, nb * _BLOCK - n))
        w = w.view(nb, _BLOCK, kb, _BLOCK)
        amax = w.abs().amax((1, 3)).clamp_min(_SMALLEST_AMAX)
        scale[e] = amax / _LARGEST
        w = (w * (_LARGEST / amax)[:, None, :, None]).clamp(-_LARGEST, _LARGEST)
        codes[e] = w.reshape(nb * _BLOCK, -1)[:n, :k].to(torch.float8_e4m3fn)
    return codes, scale


def _save_for_backward(ctx, expert_x, weight, num, padding, *more) -> None:
    """The rows are read by the weight's gradient alone and the weight by that of the rows: what no gradient reads is not kept, and may
    change.  The counts are copied: the next dispatch writes its own into the same tensor, maybe before this step's backward."""
    ctx.save_for_backward(expert_x if ctx.needs_input_grad[1] else None, weight if ctx.needs_input_grad[0] else None,
                          None if num is None else num.clone(), *more)
    ctx.shapes, ctx.expert_padding = (expert_x.shape, weight.shape), padding


def _gradients(ctx, grad_out):
    """Memory for both gradients (None: not asked for), the gradient they come from, the operands, and what else was saved.  In the place
    of an operand that was not kept stands the gradient that is as large: the calls do not read its values."""
    grad_out = grad_out.contiguous()
    if grad_out.data_ptr() % 16 != 0:   # (a part of a longer gradient may begin anywhere)
        grad_out = grad_out.clone()
    expert_x, weight, *more = ctx.saved_tensors
    grad_x = grad_out.new_zeros(ctx.shapes[0]) if ctx.needs_input_grad[0] else None
    grad_w = grad_out.new_empty(ctx.shapes[1]) if ctx.needs_input_grad[1] else None
    return grad_x, grad_w, grad_out, grad_x if expert_x is None else expert_x, grad_w if weight is None else weight, *more


class _Matmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, expert_x, weight, expert_num_tokens, expert_padding, tokens_per_expert):
        out = expert_x.new_zeros((expert_x.shape[0], weight.shape[1]))
        expert_matmul(out, expert_x, weight, expert_num_tokens, expert_padding=expert_padding,
                      tokens_per_expert=tokens_per_expert)
        _save_for_backward(ctx, expert_x, weight, expert_num_tokens, expert_padding)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        grad_x, grad_w, grad_out, expert_x, weight, num = _gradients(ctx, grad_out)
        expert_matmul_grad(grad_x, grad_w, grad_out, expert_x, weight, num, ctx.expert_padding)
        return grad_x, grad_w, None, None, None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, expert_x, weight, expert_num_tokens, expert_padding, tokens_per_expert):
        out = expert_x.new_zeros((expert_x.shape[0], weight.shape[1] // 2))
        projections = expert_x.new_empty((expert_x.shape[0], weight.shape[1]))
        expert_gated(out, expert_x, weight, expert_num_tokens, projections=projections, expert_padding=expert_padding,
                     tokens_per_expert=tokens_per_expert)
        _save_for_backward(ctx, expert_x, weight, expert_num_tokens, expert_padding, projections)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        grad_x, grad_w, grad_out, expert_x, weight, num, projections = _gradients(ctx, grad_out)
        expert_gated_grad(grad_x, grad_w, torch.empty_like(projections), grad_out, projections, expert_x, weight,
                          num, ctx.expert_padding)
        return grad_x, grad_w, None, None, None


def matmul(expert_x: torch.Tensor, weight: torch.Tensor, expert_num_tokens: Optional[torch.Tensor] = None,
           expert_padding: int = 1, tokens_per_expert: Optional[int] = None) -> torch.Tensor:
    """`expert_matmul` for autograd (bfloat16, float16); rows outside the experts' ranges are zero, and so are their
    gradients."""
    return _Matmul.apply(expert_x, weight, expert_num_tokens, expert_padding, tokens_per_expert)


def gated(expert_x: torch.Tensor, weight: torch.Tensor, expert_num_tokens: Optional[torch.Tensor] = None,
          expert_padding: int = 1, tokens_per_expert: Optional[int] = None) -> torch.Tensor:
    """`expert_gated` for autograd, as `matmul`."""
    return _Gated.apply(expert_x, weight, expert_num_tokens, expert_padding, tokens_per_expert)
