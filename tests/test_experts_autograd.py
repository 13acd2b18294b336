"""The experts' products for autograd without a GPU: plain products stand in for the library's calls.  They write past torch's
record of a tensor's versions, as the library does, and refuse what it refuses."""

import pytest
import torch

import experts_reference as ref
from pplx_garden_amd.kernels import experts


def _rows(num, padding, x, weight):
    counts = [x.shape[0]] if num is None else num.tolist()
    assert len(counts) == weight.shape[0]
    return [slice(first, first + count) for first, count in ref.ranges(counts, padding, x.shape[0])]


def _aligned(*tensors):
    for t in tensors:
        if t is not None and t.data_ptr() % 16 != 0:
            raise RuntimeError("must be multiples of 16 bytes")


def _halves(p):
    return p.double().chunk(2, -1)


@pytest.fixture(autouse=True)
def plain_calls(monkeypatch):
    def expert_matmul(out, x, w, num=None, expert_x_scale=None, weight_scale=None, expert_padding=1, tokens_per_expert=None):
        _aligned(out, x, w)
        for e, at in enumerate(_rows(num, expert_padding, x, w)):
            out.data[at] = (x[at].double() @ w[e].double().T).to(out.dtype)

    def expert_gated(out, x, w, num=None, expert_x_scale=None, weight_scale=None, out_scale=None, projections=None,
                     expert_padding=1, tokens_per_expert=None):
        expert_matmul(projections, x, w, num, expert_padding=expert_padding)
        g, u = _halves(projections)
        for at in _rows(num, expert_padding, x, w):
            out.data[at] = (ref.silu(g[at]) * u[at]).to(out.dtype)

    def expert_matmul_grad(grad_x, grad_w, grad_out, x, w, num=None, expert_padding=1):
        _aligned(grad_x, grad_w, grad_out, x, w)
        for e, at in enumerate(_rows(num, expert_padding, x, w)):
            if grad_x is not None:
                grad_x.data[at] = (grad_out[at].double() @ w[e].double()).to(grad_x.dtype)
            if grad_w is not None:
                grad_w.data[e] = (grad_out[at].double().T @ x[at].double()).to(grad_w.dtype)

    def expert_gated_grad(grad_x, grad_w, grad_projections, grad_out, projections, x, w, num=None, expert_padding=1):
        _aligned(grad_out)
        d = torch.cat(ref.gate_gradient(grad_out.double(), *_halves(projections)), -1)
        grad_projections.data.copy_(d.to(grad_projections.dtype))
        expert_matmul_grad(grad_x, grad_w, grad_projections, x, w, num, expert_padding)

    for call in (expert_matmul, expert_gated, expert_matmul_grad, expert_gated_grad):
        monkeypatch.setattr(experts, call.__name__, call)


def _layer(x, w1, w2, num):
    return experts.matmul(experts.gated(x, w1, num), w2, num)


def _operands(counts=(4, 0), n=16, k=24):
    gen = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=gen).bfloat16()

    num = torch.tensor(counts, dtype=torch.int32)
    rows = int(num.sum())
    return normal(rows, k), normal(len(counts), 2 * n, k), normal(len(counts), k, n), num, normal(rows, k)


def _gradients(x, w1, w2, num, grad_y, between=None):
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = _layer(*leaves, num)
    if between is not None:
        between()
    y.backward(grad_y)
    return [t.grad for t in leaves]


def test_backward_uses_the_counts_of_its_own_forward():
    """Dispatch writes the next step's counts into the same tensor before the first step's backward."""
    x, w1, w2, num, grad_y = _operands()
    want = _gradients(x, w1, w2, num, grad_y)
    assert (want[1][0] != 0).any() and (want[1][1] == 0).all()
    got = _gradients(x, w1, w2, num, grad_y, between=lambda: num.data.copy_(torch.tensor([0, 4])))
    assert num.tolist() == [0, 4]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_dense_product_keeps_no_counts():
    x, w1, w2, _, grad_y = _operands((4,))
    assert [g.shape for g in _gradients(x, w1, w2, None, grad_y)] == [x.shape, w1.shape, w2.shape]


@pytest.mark.parametrize("call", ["matmul", "gated"])
@pytest.mark.parametrize("frozen", ["weight", "rows"])
def test_only_what_a_gradient_needs_has_to_stay_as_it_was(call, frozen):
    """Gradients of the rows do not read the rows, nor those of a weight the weight: with one of them frozen the other's values may change
    before backward."""
    x, w1, _, num, _ = _operands((2, 3))
    grad_y = torch.randn((5, w1.shape[1] // (2 if call == "gated" else 1)), generator=torch.Generator().manual_seed(1)).bfloat16()
    grads = []
    for change in (False, True):
        rows, weight = x.clone(), w1.clone()
        (rows if frozen == "weight" else weight).requires_grad_()
        given = rows * 1                       # (a leaf that needs a gradient is not written in place)
        y = getattr(experts, call)(given, weight, num)
        if change:
            with torch.no_grad():
                (given if frozen == "weight" else weight).zero_()
        y.backward(grad_y)
        grads.append(rows.grad if frozen == "weight" else weight.grad)
    assert grads[0].float().abs().sum() > 0 and torch.equal(*grads)


@pytest.mark.parametrize("call", ["matmul", "gated"])
def test_rows_rewritten_before_backward_are_an_error(call):
    x, w1, _, num, _ = _operands((2, 3))
    given = x.clone()
    y = getattr(experts, call)(given, w1.requires_grad_(), num)
    given.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("call", ["matmul", "gated"])
def test_a_gradient_that_autograd_cuts_out_of_a_longer_one(call):
    """The result flattened behind a few other values: its gradient is whole rows, but begins at any multiple of two bytes."""
    x, w1, _, num, _ = _operands((2, 3))
    grads = []
    for joined in (False, True):
        rows, weight = x.clone().requires_grad_(), w1.clone().requires_grad_()
        y = getattr(experts, call)(rows, weight, num)
        c = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).bfloat16()
        if joined:
            torch.cat([y.new_zeros(3), y.flatten()]).backward(torch.cat([c.new_zeros(3), c.flatten()]))
        else:
            y.backward(c)
        grads.append((rows.grad, weight.grad))
    for a, b in zip(*grads):
        assert a.float().abs().sum() > 0 and torch.equal(a, b)


def test_quantized_parameters_keep_no_graph():
    """A model's weights are parameters: their codes are constants, and the float copies behind them are gone."""
    weight = torch.nn.Parameter(_operands()[1].float())
    codes, scale = experts.quantize_weight(weight)
    for t in (codes, scale):
        assert not t.requires_grad and t.grad_fn is None
    for got, want in zip((codes, scale), experts.quantize_weight(weight.detach())):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
