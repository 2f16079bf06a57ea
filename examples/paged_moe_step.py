"""One sparsely routed layer over a paged batch, with its training step.

    python examples/paged_moe_step.py

1. DeviceBlockTable gives the tokens of a mixed batch (prompts and single
   tokens, padded to a fixed capacity) their pages, slots and positions.
2. DeviceRouter chooses each token's experts; the padding that step 1 marked is
   left out of the counts and the balance loss.
3. DeviceDispatch groups the tokens' rows by expert, the experts' products run
   on the groups, and Combine sums them back.
4. The gradients run the same way back, and a few steps of gradient descent
   fit the layer to a target while the balance loss keeps the counts together.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "luisacompute-parallelprimitive_b200"))
import lcpp_b200 as L  # noqa: E402

I32 = {"dtype": torch.int32, "device": "cuda"}
F32 = {"dtype": torch.float32, "device": "cuda"}


def lay_out(context, new, capacity, block=16, width=64):
    """Slots, positions and requests of the step's tokens, and the extended table."""
    n = context.numel()
    pages = torch.randperm(n * width + capacity, device="cuda").to(torch.int32)
    table, free = pages[:n * width].view(n, width).clone(), pages[n * width:].contiguous()
    out = {"table": table, "used": torch.zeros(1, **I32), "seq_lens": torch.zeros(n, **I32),
           "starts": torch.zeros(n + 1, **I32), "slots": torch.zeros(capacity, dtype=torch.int64, device="cuda"),
           "positions": torch.zeros(capacity, **I32), "requests": torch.zeros(capacity, **I32)}
    temp = L.alloc_temp(L.DeviceBlockTable.GetTempStorageBytes(n, capacity))
    L.DeviceBlockTable().Extend(temp, context, new, table, free, None, out["used"], out["seq_lens"], out["starts"],
                                out["slots"], out["positions"], out["requests"], n, block)
    return out


class Layer:
    """Router and experts of one layer, and the buffers a step of `tokens` tokens needs."""

    def __init__(self, tokens, hidden, experts, top_k, align=16, dtype=torch.bfloat16):
        self.t, self.h, self.e, self.k, self.align = tokens, hidden, experts, top_k, align
        self.router = torch.randn(hidden, experts, **F32) / hidden ** 0.5
        self.experts = torch.randn(experts, hidden, hidden, **F32) / hidden ** 0.5
        rows = L.DeviceDispatch.MaxRows(tokens, top_k, experts, align)
        self.temp = L.alloc_temp(max(L.DeviceRouter.GetTempStorageBytes(tokens, experts),
                                     L.DeviceDispatch.GetTempStorageBytes(tokens, top_k, experts)))
        self.weights, self.chosen = torch.zeros(tokens, top_k, **F32), torch.zeros(tokens, top_k, **I32)
        self.counts, self.routed, self.loss = torch.zeros(experts, **I32), torch.zeros(1, **I32), torch.zeros(1, **F32)
        self.starts, self.row_of = torch.zeros(experts + 1, **I32), torch.zeros(tokens, top_k, **I32)
        self.pair_of = torch.zeros(rows, **I32)
        self.rows, self.grad_rows = (torch.zeros(rows, hidden, dtype=dtype, device="cuda") for _ in range(2))
        self.grad_weights = torch.zeros(tokens, top_k, **F32)
        self.options = {"score": L.SCORE_SOFTMAX, "renormalize": True, "weight_scale": 1.0, "loss_coef": 1.0}

    def segments(self):
        starts = self.starts.tolist()
        return [(e, starts[e], starts[e + 1]) for e in range(self.e) if starts[e] < starts[e + 1]]

    def forward(self, x, requests):
        self.x = x
        self.logits = (x.float() @ self.router).to(x.dtype)
        L.DeviceRouter().Forward(self.temp, self.logits, self.weights, self.chosen, self.counts, self.routed,
                                 self.loss, self.t, self.e, self.k, d_token_request=requests, **self.options)
        d = L.DeviceDispatch()
        d.Plan(self.temp, self.chosen, self.starts, self.row_of, self.pair_of, self.t, self.k, self.e, self.align)
        d.Gather(x, self.row_of, self.pair_of, self.starts, self.rows, self.t, self.k, self.e)
        self.products = torch.zeros_like(self.rows)
        for e, a, b in self.segments():
            self.products[a:b] = self.rows[a:b] @ self.experts[e].to(x.dtype)
        out = torch.empty_like(x)
        d.Combine(self.products, self.row_of, self.weights, out, self.t, self.k)
        return out

    def backward(self, grad_out, balance):
        """Gradients of sum(out * grad_out) + balance * loss: (router, experts, x)."""
        d = L.DeviceDispatch()
        d.CombineBackward(grad_out, self.products, self.row_of, self.pair_of, self.starts, self.weights,
                          self.grad_rows, self.grad_weights, self.t, self.k, self.e)
        grad_experts, grad_in = torch.zeros_like(self.experts), torch.zeros_like(self.rows)
        for e, a, b in self.segments():
            grad_experts[e] = self.rows[a:b].float().t() @ self.grad_rows[a:b].float()
            grad_in[a:b] = self.grad_rows[a:b] @ self.experts[e].to(grad_in.dtype).t()
        grad_x = torch.empty_like(self.x)
        d.Combine(grad_in, self.row_of, None, grad_x, self.t, self.k)  # Gather's gradient
        grad_logits = torch.empty_like(self.logits)
        L.DeviceRouter().Backward(self.logits, self.chosen, self.counts, self.routed, self.grad_weights,
                                  torch.full((1,), balance, **F32), grad_logits, self.t, self.e, self.k,
                                  **self.options)
        grad_router = self.x.float().t() @ grad_logits.float()
        return grad_router, grad_experts, grad_x.float() + grad_logits.float() @ self.router.t()


def main(steps=30):
    torch.manual_seed(0)
    capacity, hidden, experts, top_k = 512, 64, 8, 2
    context = torch.tensor([0, 200, 17, 0, 90, 33], **I32)
    new = torch.tensor([250, 1, 1, 180, 1, 40], **I32)
    step = lay_out(context, new, capacity)
    tokens = int(step["starts"][-1])
    live = step["requests"] >= 0
    print(f"{tokens} tokens of {context.numel()} requests in {int(step['used'])} new pages, {capacity} entries")

    layer = Layer(capacity, hidden, experts, top_k)
    x = torch.randn(capacity, hidden, **F32).to(torch.bfloat16)
    target = torch.tanh(x.float() @ torch.randn(hidden, hidden, **F32) / hidden ** 0.5)
    first = last = None
    for i in range(steps):
        out = layer.forward(x, step["requests"])
        error = torch.where(live[:, None], out.float() - target, 0)
        fit = float((error ** 2).sum() / tokens)
        grad_router, grad_experts, _ = layer.backward((2 * error / tokens).to(x.dtype), balance=1.0)
        layer.router -= 0.3 * grad_router
        layer.experts -= 0.3 * grad_experts
        last = (fit, float(layer.loss), layer.counts.tolist())
        first = first or last
    print("first step: fit %.3f, balance %.4f, tokens per expert %s" % first)
    print("last step:  fit %.3f, balance %.4f, tokens per expert %s" % last)
    assert sum(last[2]) == tokens * top_k and last[0] < first[0]
    return first, last


if __name__ == "__main__":
    main()
