"""Buffers that steps share: what the calls write is known to autograd, and a backward pass that would read rows of another step is
refused."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "pplx-garden_amd" / "examples" / "moe_layer.py"
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def device():
    return torch.device("cuda", torch.cuda.current_device())


def _changed(tensors, call):
    """Names of the tensors whose versions a call raises."""
    before = {name: t._version for name, t in tensors.items()}
    call()
    torch.cuda.synchronize()
    return {name for name, t in tensors.items() if t._version != before[name]}


@pytest.fixture(params=[True, False], ids=["fp8", "bf16"])
def layer(request):
    example = _example()
    a = example.parse(["--tokens", "8", "--hidden", "256", "--inter", "128", "--experts", "4", "--topk", "2", "--ranks", "2"])
    ranks, _, _ = example.make_layer(a, device(), fp8=request.param)
    yield example, ranks
    for k in ranks:
        k["op"].destroy()


def _dispatch(k, **halves):
    k["op"].dispatch(out_expert_num_tokens=k["num"], out_expert_x=k["rows"], out_expert_x_scale=k["scale"], dp_x=k["x"],
                     dp_x_scale=None, indices=k["indices"], weights=k["weights"], **halves)


def _combine(k, **halves):
    k["op"].combine(out_tokens=k["out"], indices=k["indices"], weights=k["weights"], expert_y=k["y"], **halves)


def test_dispatch_and_combine_raise_the_versions_of_what_they_write(layer):
    example, ranks = layer
    tensors = {f"{name}{r}": t for r, k in enumerate(ranks) for name, t in k.items() if isinstance(t, torch.Tensor)}
    received = {f"{name}{r}" for r in range(2) for name in ("num", "rows", "scale") if f"{name}{r}" in tensors}
    # a collective runs, and writes, when the last rank has made the call
    assert _changed(tensors, lambda: _dispatch(ranks[0])) == set()
    assert _changed(tensors, lambda: _dispatch(ranks[1])) == received
    assert _changed(tensors, lambda: _combine(ranks[0])) == set()
    assert _changed(tensors, lambda: _combine(ranks[1])) == {"out0", "out1"}
    for k in ranks:
        assert _changed(tensors, lambda: _dispatch(k, do_recv=False)) == set()
    for r, k in enumerate(ranks):
        assert _changed(tensors, lambda: _dispatch(k, do_send=False)) == {n for n in received if n.endswith(str(r))}
    for k in ranks:
        assert _changed(tensors, lambda: _combine(k, do_recv=False)) == set()
    for r, k in enumerate(ranks):
        assert _changed(tensors, lambda: _combine(k, do_send=False)) == {f"out{r}"}


def test_the_products_raise_the_versions_of_what_they_write():
    from pplx_garden_amd.kernels import experts
    n, k, rows = 16, 32, 6
    num = torch.tensor([2, 4], dtype=torch.int32, device=device())

    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=device())

    t = dict(x=zeros(rows, k), w=zeros(2, 2 * n, k), y=zeros(rows, 2 * n), h=zeros(rows, n), p=zeros(rows, 2 * n),
             dh=zeros(rows, n), dp=zeros(rows, 2 * n), dx=zeros(rows, k), dw=zeros(2, 2 * n, k), num=num)
    assert _changed(t, lambda: experts.expert_matmul(t["y"], t["x"], t["w"], num)) == {"y"}
    assert _changed(t, lambda: experts.expert_gated(t["h"], t["x"], t["w"], num)) == {"h"}
    assert _changed(t, lambda: experts.expert_gated(t["h"], t["x"], t["w"], num, projections=t["p"])) == {"h", "p"}
    assert _changed(t, lambda: experts.expert_gated_grad(t["dx"], t["dw"], t["dp"], t["dh"], t["p"], t["x"], t["w"], num)) == {
        "dx", "dw", "dp"}
    assert _changed(t, lambda: experts.expert_matmul_grad(t["dx"], None, t["y"], t["x"], t["w"], num)) == {"dx"}
    assert _changed(t, lambda: experts.expert_matmul_grad(None, t["dw"], t["y"], t["x"], t["w"], num)) == {"dw"}
    f8 = dict(x=zeros(rows, k, dtype=torch.float8_e4m3fn), xs=zeros(rows, 1, dtype=torch.float32),
              w=zeros(2, 2 * n, k, dtype=torch.float8_e4m3fn), ws=zeros(2, 1, 1, dtype=torch.float32),
              h=zeros(rows, n, dtype=torch.float8_e4m3fn), hs=zeros(rows, 1, dtype=torch.float32), y=zeros(rows, 2 * n), num=num)
    scales = dict(expert_x_scale=f8["xs"], weight_scale=f8["ws"])
    assert _changed(f8, lambda: experts.expert_matmul(f8["y"], f8["x"], f8["w"], num, **scales)) == {"y"}
    assert _changed(f8, lambda: experts.expert_gated(f8["h"], f8["x"], f8["w"], num, out_scale=f8["hs"], **scales)) == {"h", "hs"}


def test_inference_tensors_have_no_versions():
    from pplx_garden_amd.kernels.experts import expert_matmul
    with torch.inference_mode():
        x, w = torch.ones((3, 16), device=device()).bfloat16(), torch.ones((1, 8, 16), device=device()).bfloat16()
        inside = torch.zeros((3, 8), device=device()).bfloat16()
        expert_matmul(inside, x, w)
    outside = torch.zeros((3, 8), device=device()).bfloat16()
    expert_matmul(inside, x, w)
    expert_matmul(outside, x, w)
    with torch.inference_mode():
        expert_matmul(outside, x, w)
    assert (inside == 16).all() and (outside == 16).all()


@pytest.mark.parametrize("layer", [False], ids=["bf16"], indirect=True)
def test_a_second_dispatch_into_the_rows_of_a_pending_backward_is_found_out(layer):
    """Two microbatches through one receive buffer, both forward before the first one's backward."""
    from pplx_garden_amd.kernels.experts import gated, matmul
    example, ranks = layer

    def forward(k):
        x = k["rows"].detach().requires_grad_()
        return x, matmul(gated(x, k["up"], k["num"]), k["down"], k["num"])

    k = ranks[0]
    example.dispatch(ranks)
    x, y = forward(k)
    y.backward(torch.ones_like(y))             # in time
    want = [g.clone() for g in (x.grad, k["up"].grad, k["down"].grad)]
    first = forward(k)[1]
    for other in ranks:
        other["x"] = -other["x"]
    example.dispatch(ranks)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        first.backward(torch.ones_like(first))

    # with rows of its own, and the counts shared, the first step's gradients are what they were
    for other in ranks:
        other["x"] = -other["x"]
    example.dispatch(ranks)
    k["up"].grad = k["down"].grad = None
    x, y = forward(k)
    k["rows"] = torch.zeros_like(k["rows"])
    for other in ranks:
        other["indices"] = (3 - other["indices"].view(torch.int32)).view(torch.uint32).contiguous()
    counts = k["num"].clone()
    example.dispatch(ranks)
    assert not torch.equal(counts, k["num"])
    y.backward(torch.ones_like(y))
    for got, expected in zip((x.grad, k["up"].grad, k["down"].grad), want):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("call", ["matmul", "gated"])
def test_a_gradient_that_begins_at_any_address(call):
    """autograd hands over a part of a longer gradient: whole rows, behind three other values."""
    from pplx_garden_amd.kernels import experts
    gen = torch.Generator(device=device())
    gen.manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device()).bfloat16()

    x, w, num = normal(5, 24), normal(2, 32, 24), torch.tensor([2, 3], dtype=torch.int32, device=device())
    c = normal(5, 32 if call == "matmul" else 16)
    grads = []
    for joined in (False, True):
        rows, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = getattr(experts, call)(rows, weight, num)
        if joined:
            torch.cat([y.new_zeros(3), y.flatten()]).backward(torch.cat([c.new_zeros(3), c.flatten()]))
        else:
            y.backward(c)
        grads.append((rows.grad, weight.grad))
    for a, b in zip(*grads):
        assert a.float().abs().sum() > 0 and torch.equal(a, b)


def test_a_hint_of_no_rows_is_one_of_the_fewest():
    from pplx_garden_amd.kernels.experts import expert_gated, expert_matmul
    gen = torch.Generator(device=device())
    gen.manual_seed(4)
    x, w = (torch.randn(s, generator=gen, device=device()).bfloat16() for s in ((40, 64), (4, 32, 64)))
    num = torch.tensor([0, 1, 0, 2], dtype=torch.int32, device=device())
    got = []
    for expected in (0, 1):
        y, h = (torch.zeros((40, n), device=device()).bfloat16() for n in (32, 16))
        expert_matmul(y, x, w, num, tokens_per_expert=expected)
        expert_gated(h, x, w, num, tokens_per_expert=expected)
        got.append((y, h))
    for a, b in zip(*got):
        assert a.float().abs().sum() > 0 and torch.equal(a, b)


@pytest.mark.parametrize("arguments", [[], ["--padding", "16", "--tokens", "37", "--inter", "264"]])
def test_the_gradients_of_the_examples_training_step(arguments):
    """Of the rows and of both weights, rank by rank, against the layer's derivative in 64 bits on the rows that dispatch has left.  Every rounding
    to bfloat16 is one of 2^-8 at most: gates, ups, the gradient of the block, that of the projections and the result of the rows and of the
    first weights; the block and the result of the second weights."""
    import experts_reference as ref
    example = _example()
    a = example.parse(["--train", *arguments])
    ranks, _, _ = example.make_layer(a, device(), fp8=False)
    gen = torch.Generator(device=device())
    gen.manual_seed(5)
    grad_y = [torch.randn(k["y"].shape, generator=gen, device=device()).bfloat16() for k in ranks]
    example.train(a, ranks, grad_y)
    for k, c in zip(ranks, grad_y):
        rows, up, down = (t.detach().double() for t in (k["rows"], k["up"], k["down"]))
        got = dict(rows=k["grad_rows"], up=k["up"].grad, down=k["down"].grad)
        want = dict(rows=torch.zeros_like(rows), up=torch.zeros_like(up), down=torch.zeros_like(down))
        for e, (first, count) in enumerate(ref.ranges(k["num"].tolist(), a.padding, rows.shape[0])):
            at = slice(first, first + count)
            g, u = (rows[at] @ up[e].T).chunk(2, -1)
            dy = c[at].double()
            want["down"][e] = dy.T @ (ref.silu(g) * u)
            d = torch.cat(ref.gate_gradient(dy @ down[e], g, u), -1)
            want["rows"][at], want["up"][e] = d @ up[e], d.T @ rows[at]
        for name, roundings in (("rows", 5), ("up", 5), ("down", 2)):
            off = (got[name].double() - want[name]).norm() / want[name].norm()
            assert off < roundings * 2.0 ** -8, (name, off.item())
        assert not got["rows"][want["rows"].abs().sum(1) == 0].any()
        assert not got["up"][k["num"] == 0].any() and not got["down"][k["num"] == 0].any()
        k["op"].destroy()


@pytest.mark.parametrize("call", ["matmul", "gated"])
def test_gradients_with_the_rows_or_the_weight_frozen(call):
    """The operand that is not read is not kept, and may have changed by then; no rows at all are a gradient of zeros."""
    from pplx_garden_amd.kernels import experts
    gen = torch.Generator(device=device())
    gen.manual_seed(6)
    x, w = (torch.randn(s, generator=gen, device=device()).bfloat16() for s in ((300, 72), (3, 48, 72)))
    num = torch.tensor([100, 0, 200], dtype=torch.int32, device=device())
    c = torch.randn((300, 48 if call == "matmul" else 24), generator=gen, device=device()).bfloat16()

    product = getattr(experts, call)
    rows, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
    product(rows, weight, num).backward(c)
    want = rows.grad, weight.grad
    assert all(g.float().abs().sum() > 0 for g in want)
    weight = w.clone().requires_grad_()
    product(x, weight, num).backward(c)
    assert torch.equal(weight.grad, want[1])
    rows = x.clone().requires_grad_()
    given = rows * 1
    y = product(given, w, num)
    experts.expert_matmul(given.detach(), c.new_zeros((300, 8)), c.new_zeros((3, 72, 8)), num)   # writes the rows again
    assert not given.any()
    y.backward(c)
    assert torch.equal(rows.grad, want[0])
    weight.grad = None
    product(x[:0], weight, torch.zeros_like(num)).backward(c[:0])
    assert weight.grad.shape == w.shape and not weight.grad.any()
