"""A mixture-of-experts layer on one GPU: dispatch, the experts' gated blocks, combine.

    python pplx-garden_amd/examples/moe_layer.py [--tokens 128] [--hidden 2048] [--inter 768] [--experts 32] [--topk 4]
                                                 [--ranks 4] [--train]

Serving (the default): tokens are dispatched as e4m3 rows with a scale per 128 entries, `expert_gated` reads them and writes e4m3
rows again, `expert_matmul` reads those and writes what `combine` gathers.  Training (`--train`): the same layer on bfloat16
rows with gradients of the experts' weights and of their rows.  Prints how far the layer's result is from the same layer
in float and what a step takes.
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from pplx_garden_amd.distributed.loopback import LoopbackWorld  # noqa: E402
from pplx_garden_amd.kernels import experts as ffn  # noqa: E402
from pplx_garden_amd.kernels.p2p_all_to_all import P2PAllToAll  # noqa: E402


def make_layer(a, device, fp8):
    """Operators and buffers of every rank, and the experts' weights (as the model's, and as its ranks keep them)."""
    world = LoopbackWorld(a.ranks, device=device)
    local = a.experts // a.ranks
    row_dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    ops = [P2PAllToAll(max_num_tokens=a.tokens, num_experts=a.experts, expert_padding=a.padding, hidden_dim=a.hidden,
                       hidden_dim_scale=a.hidden // 128 if fp8 else None, in_dtype=row_dtype, out_dtype=torch.bfloat16,
                       scale_dtype=torch.float32 if fp8 else None, num_experts_per_token=a.topk, device=device,
                       global_group=world.group(r)) for r in range(a.ranks)]
    gen = torch.Generator(device=device)
    gen.manual_seed(a.seed)
    up = torch.randn((a.experts, 2 * a.inter, a.hidden), generator=gen, device=device) * a.hidden ** -0.5
    down = torch.randn((a.experts, a.hidden, a.inter), generator=gen, device=device) * a.inter ** -0.5
    tokens = [torch.randn((a.tokens, a.hidden), generator=gen, device=device).bfloat16() for _ in range(a.ranks)]
    scores = [torch.randn((a.tokens, a.experts), generator=gen, device=device) for _ in range(a.ranks)]
    routes = [s.topk(a.topk, dim=-1) for s in scores]
    rows = a.ranks * a.tokens * a.topk + local * (a.padding - 1)   # all copies could reach one rank
    ranks = []
    for r in range(a.ranks):
        mine = slice(r * local, (r + 1) * local)
        rank = dict(op=ops[r], x=tokens[r], indices=routes[r].indices.int().view(torch.uint32),
                    weights=torch.softmax(routes[r].values, -1).contiguous(),
                    num=torch.zeros(local, dtype=torch.int32, device=device),
                    rows=torch.zeros((rows, a.hidden), dtype=row_dtype, device=device),
                    y=torch.zeros((rows, a.hidden), dtype=torch.bfloat16, device=device),
                    out=torch.zeros((a.tokens, a.hidden), dtype=torch.bfloat16, device=device))
        if fp8:
            rank["up"], rank["up_scale"] = ffn.quantize_weight(up[mine])
            rank["down"], rank["down_scale"] = ffn.quantize_weight(down[mine])
            rank.update(scale=torch.zeros((rows, a.hidden // 128), device=device),
                        h=torch.zeros((rows, a.inter), dtype=torch.float8_e4m3fn, device=device),
                        h_scale=torch.zeros((rows, -(-a.inter // 128)), device=device))
        else:
            rank["up"], rank["down"] = (w[mine].bfloat16().requires_grad_() for w in (up, down))
            rank["scale"] = None
        ranks.append(rank)
    return ranks, up, down


def dispatch(ranks):
    for k in ranks:
        k["op"].dispatch(out_expert_num_tokens=k["num"], out_expert_x=k["rows"], out_expert_x_scale=k["scale"], dp_x=k["x"],
                         dp_x_scale=None, indices=k["indices"], weights=k["weights"])


def combine(ranks):
    for k in ranks:
        k["op"].combine(out_tokens=k["out"], indices=k["indices"], weights=k["weights"], expert_y=k["y"])


def serve(a, ranks):
    """One layer of serving: nothing in it waits for the GPU or asks it for counts."""
    expected = max(1, a.ranks * a.tokens * a.topk // a.experts)
    dispatch(ranks)
    for k in ranks:
        rows = dict(expert_num_tokens=k["num"], expert_padding=a.padding, tokens_per_expert=expected)
        ffn.expert_gated(k["h"], k["rows"], k["up"], expert_x_scale=k["scale"], weight_scale=k["up_scale"],
                         out_scale=k["h_scale"], **rows)
        ffn.expert_matmul(k["y"], k["h"], k["down"], expert_x_scale=k["h_scale"], weight_scale=k["down_scale"], **rows)
    combine(ranks)


def train(a, ranks, grad_y):
    """The same with gradients: `grad_y` is what the loss makes of every rank's expert rows.  The products read the receive buffer itself, so
    backward comes before the next dispatch into it (which would make it raise)."""
    dispatch(ranks)
    for k, g in zip(ranks, grad_y):
        x = k["rows"].detach().requires_grad_()
        y = ffn.matmul(ffn.gated(x, k["up"], k["num"], a.padding), k["down"], k["num"], a.padding)
        k["y"] = y.detach()
        k["up"].grad = k["down"].grad = None
        y.backward(g)
        k["grad_rows"] = x.grad
    combine(ranks)


def in_float(a, ranks, up, down):
    """The layer token by token, expert by expert, in 32 bits."""
    outs = []
    for k in ranks:
        x, out = k["x"].float(), torch.zeros((a.tokens, a.hidden), device=up.device)
        index = k["indices"].view(torch.int32).long()
        for e in range(a.experts):
            token, place = (index == e).nonzero(as_tuple=True)
            if token.numel() == 0:
                continue
            gate, rise = (x[token] @ up[e].T).chunk(2, -1)
            y = (torch.nn.functional.silu(gate) * rise) @ down[e].T
            out.index_add_(0, token, y * k["weights"][token, place, None])
        outs.append(out)
    return torch.cat(outs)


def parse(arguments=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 128), ("hidden", 2048), ("inter", 768), ("experts", 32), ("topk", 4), ("ranks", 4), ("padding", 1),
                        ("steps", 20), ("seed", 0)):
        p.add_argument(f"--{name}", type=int, default=value)
    p.add_argument("--train", action="store_true")
    return p.parse_args(arguments)


def main(arguments=None) -> float:
    """Runs the layer; returns its distance from the layer in float, in 2-norms."""
    a = parse(arguments)
    device = torch.device("cuda", torch.cuda.current_device())
    ranks, up, down = make_layer(a, device, fp8=not a.train)
    grad_y = [torch.randn(k["y"].shape, device=device).bfloat16() for k in ranks] if a.train else None

    def step():
        return train(a, ranks, grad_y) if a.train else serve(a, ranks)

    step()
    torch.cuda.synchronize()
    want, got = in_float(a, ranks, up, down), torch.cat([k["out"] for k in ranks]).float()
    off = ((got - want).norm() / want.norm()).item()
    begin = time.perf_counter()
    for _ in range(a.steps):
        step()
    torch.cuda.synchronize()
    took = (time.perf_counter() - begin) / max(1, a.steps)
    print(f"{'training' if a.train else 'serving'}: {a.ranks} ranks x {a.tokens} tokens, {a.experts} experts, top {a.topk}, hidden {a.hidden}, "
          f"inter {a.inter}: {off:.4f} from the layer in float, {took * 1e6:.1f} us a step", flush=True)
    for k in ranks:
        k["op"].destroy()
    return off


if __name__ == "__main__":
    main()
