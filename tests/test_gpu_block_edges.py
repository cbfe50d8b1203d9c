"""The block operators (ascq_add_rms_norm_quant, ascq_quant_linear, ascq_moe_*) at the edges of their ranges: streams beside each
other, infinities, tiny and empty rows, very many rows.  Each test states its tolerance."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_side_stream_beside_work_on_the_current_one(ascq_gpu):
    """Calls on a stream while the current one still writes to blocks it has given back: the calls' own memory is none of those
    (whole numbers, equal bits)"""
    a = ascq_gpu
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn(40, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
    w = (torch.randn(640, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
    xs, ws = torch.rand(40, generator=g, device="cuda"), torch.rand(640, generator=g, device="cuda")
    logits = torch.randn(3000, 64, generator=g, device="cuda")
    linear = lambda st: a.quant_linear(x, xs, w, ws, out_dtype=torch.float32, stream=st)  # noqa: E731
    want, route = linear(None), a.moe_route(logits, 6)
    need = a.quant_linear_workspace_size(x, w, True, torch.float32)
    assert need > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for st in (side, side.cuda_stream):
        for _ in range(5):
            for size in (need, want.numel() * 4, 3000 * 6 * 4, 64 * 47 * 8):
                given_back = torch.empty(size, dtype=torch.uint8, device="cuda")
                for _ in range(30):
                    given_back.fill_(255)
                del given_back
            got, r = linear(st), a.moe_route(logits, 6, stream=st)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert all(torch.equal(p, q) for p, q in zip(r, route))


def test_route_gradient_of_a_large_upstream_gradient(ascq_gpu):
    """grad_loss E counts / (sum counts routed) in an order that does not pass fp32's range while the result is inside it: the
    gradient of 2e38 is 2^100 times that of 2e38 / 2^100, bit for bit (a power of two; nothing here is subnormal)"""
    a = ascq_gpu
    x = torch.randn(40, 16, generator=torch.Generator().manual_seed(3)).cuda()
    r = a.moe_route(x, 2)
    grad = lambda v: a.moe_route_grad(x, r.weights, r.experts, r.counts, r.routed,  # noqa: E731
                                      grad_loss=torch.tensor([v], device="cuda"))
    large, small = grad(2e38), grad(2e38 / 2.0 ** 100)
    assert torch.isfinite(large).all() and torch.equal(large, small * 2.0 ** 100)
