"""A quantised mixture-of-experts block: residual + RMS norm to int8, an int8 router, routed experts and a shared one.

    python examples/quantized_moe_block.py [--tokens 4096] [--hidden 4096] [--ffn 1408] [--experts 16] [--top-k 2]

Every tensor operation of the forward pass is one of the library's: add_rms_norm_quant, quant_linear (router, shared
expert), moe_route, moe_dispatch, quant_group_matmul (routed experts), quant_dynamic_per_token and moe_combine.  The
command runs a batch of tokens and one decode step, compares both with the same block in fp32, takes the router's gradient
of a loss on the output plus the balance loss, and prints the errors and the times.  Weights and inputs are random.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "asc-devkit_clone_amd"))
import ascq  # noqa: E402


def quantize_weight(w: torch.Tensor):
    """[..., out, in] -> int8 codes and one fp32 scale per output channel"""
    scale = w.abs().amax(dim=-1) / 127
    return (w / scale[..., None]).round().to(torch.int8).contiguous(), scale.contiguous()


class QuantizedMoEBlock:
    """weights: dict of fp32 tensors -- gamma [H], router [E, H], up [E, F, H], down [E, H, F], shared_up [S, H],
    shared_down [H, S]"""

    def __init__(self, weights: dict, top_k: int, eps: float = 1e-6):
        self.top_k, self.eps = top_k, eps
        self.gamma = weights["gamma"].to(torch.bfloat16)
        for name in ("router", "up", "down", "shared_up", "shared_down"):
            setattr(self, name, quantize_weight(weights[name]))

    def forward(self, x: torch.Tensor, residual: torch.Tensor):
        """x, residual [tokens, H] bf16 -> the new residual stream, and what the router's gradient needs"""
        q, scale, h = ascq.add_rms_norm_quant(x, self.gamma, self.eps, residual=residual)
        logits = ascq.quant_linear(q, scale, *self.router, out_dtype=torch.float32)
        routing = ascq.moe_route(logits, self.top_k)
        rows, row_scale = ascq.moe_dispatch(q, scale, routing.slots, routing.tokens)
        mid = ascq.quant_group_matmul(rows, row_scale, *self.up, routing.counts, list_type=1, w_trans=True,
                                      activation=ascq.ACT_FASTER_GELU)
        y = ascq.quant_group_matmul(*ascq.quant_dynamic_per_token(mid), *self.down, routing.counts, list_type=1, w_trans=True)
        out = ascq.moe_combine(y, routing.slots, routing.weights, residual=h)
        shared = ascq.quant_linear(q, scale, *self.shared_up, activation=ascq.ACT_FASTER_GELU)
        ascq.quant_linear(*ascq.quant_dynamic_per_token(shared), *self.shared_down, residual=out, out=out)
        return out, (logits, routing, y)

    def router_gradient(self, saved, grad_out: torch.Tensor, balance: float):
        """d / d logits of a loss whose gradient at the output is grad_out, plus balance times the balance loss"""
        logits, routing, y = saved
        grad_weights, _ = ascq.moe_combine_grad(grad_out, y, routing.slots, routing.tokens, routing.weights, need_grad_y=False)
        return ascq.moe_route_grad(logits, routing.weights, routing.experts, routing.counts, routing.routed,
                                   grad_weights=grad_weights, grad_loss=torch.full((1,), balance, device=logits.device))


def reference(weights: dict, top_k: int, experts: torch.Tensor, logits: torch.Tensor, x, residual, eps: float = 1e-6):
    """the block in fp32 with the given choices of experts and logits"""
    h = (x.float() + residual.float()).to(x.dtype).float()
    n = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + eps) * weights["gamma"].to(torch.bfloat16).float()
    p = torch.softmax(logits, dim=1).gather(1, experts.long())
    p = p / p.sum(dim=1, keepdim=True)
    gelu = lambda v: v * torch.sigmoid(1.702 * v)  # noqa: E731
    out = h + gelu(n @ weights["shared_up"].t()) @ weights["shared_down"].t()
    for e in range(weights["up"].shape[0]):
        t, j = (experts == e).nonzero(as_tuple=True)
        if t.numel():
            out.index_add_(0, t, p[t, j, None] * (gelu(n[t] @ weights["up"][e].t()) @ weights["down"][e].t()))
    return out


def random_weights(hidden: int, ffn: int, experts: int, shared: int, device="cuda"):
    g = torch.Generator(device=device).manual_seed(0)
    w = lambda *s: torch.randn(s, generator=g, device=device) / s[-1] ** 0.5  # noqa: E731
    return dict(gamma=1 + 0.1 * torch.randn(hidden, generator=g, device=device), router=w(experts, hidden),
                up=w(experts, ffn, hidden), down=w(experts, hidden, ffn), shared_up=w(shared, hidden),
                shared_down=w(hidden, shared))


def run(tokens: int, hidden: int, ffn: int, experts: int, top_k: int):
    """relative error of the block against fp32, the balance loss and the router's gradient"""
    weights = random_weights(hidden, ffn, experts, ffn)
    block = QuantizedMoEBlock(weights, top_k)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, residual, grad = (torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    out, saved = block.forward(x, residual)
    want = reference(weights, top_k, saved[1].experts, saved[0], x, residual)
    delta = want - (x.float() + residual.float())  # (what the block adds to the stream)
    err = ((out.float() - want).norm() / delta.norm()).item()
    gradient = block.router_gradient(saved, grad, 0.01)
    return block, (x, residual), err, saved[1].loss.item(), gradient


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("tokens", 4096), ("hidden", 4096), ("ffn", 1408), ("experts", 16), ("top-k", 2)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    for tokens in (a.tokens, 1):
        block, inputs, err, loss, gradient = run(tokens, a.hidden, a.ffn, a.experts, a.top_k)
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for _ in range(3):
            block.forward(*inputs)
        start.record()
        for _ in range(20):
            block.forward(*inputs)
        stop.record()
        torch.cuda.synchronize()
        print(f"{tokens} tokens: {start.elapsed_time(stop) / 20 * 1e3:.0f} us, error {err:.4f} of what the block adds, "
              f"balance loss {loss:.3f}, router gradient {gradient.norm().item():.3g}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
