"""An attention layer that answers from a paged cache of bounded size, and its training step.

    python examples/paged_cache_decode.py

1. DeviceBlockTable gives a step's tokens (prompts first, then one token for each request) their
   pages, slots and positions.
2. DeviceRotary turns queries and keys by their positions and writes keys and values to their slots.
3. DevicePagedAttention attends from each request's last token over its pages, and adds up how much
   attention every cached token got.
4. When requests have grown past their budget, DeviceCacheEviction chooses the tokens that got least,
   moves the others together and gives pages back to the free list that step 1 takes them from.
5. In training, where no cache is kept, the same layer runs over whole sequences; DeviceRotary's
   Backward takes the gradients of the turned queries and keys back.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "luisacompute-parallelprimitive_b200"))
import lcpp_b200 as L  # noqa: E402

I32 = {"dtype": torch.int32, "device": "cuda"}
F32 = {"dtype": torch.float32, "device": "cuda"}


class Rotated(torch.autograd.Function):
    """DeviceRotary as a differentiable function of queries and keys [tokens, heads, dim]."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies):
        ctx.positions, ctx.frequencies = positions, frequencies
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        L.DeviceRotary().Forward(q, k, q_out, k_out, positions, frequencies, q.shape[0])
        return q_out, k_out

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        grad_q, grad_k = grad_q.contiguous(), grad_k.contiguous()
        q_out, k_out = torch.empty_like(grad_q), torch.empty_like(grad_k)
        L.DeviceRotary().Backward(grad_q, grad_k, q_out, k_out, ctx.positions, ctx.frequencies, grad_q.shape[0])
        return q_out, k_out, None, None


class Layer:
    """Projections and the frequencies of one attention layer."""

    def __init__(self, hidden=128, heads=8, kv_heads=2, dim=32, dtype=torch.bfloat16):
        self.heads, self.kv_heads, self.dim, self.dtype = heads, kv_heads, dim, dtype
        width = (heads + 2 * kv_heads) * dim
        self.qkv = (torch.randn(hidden, width, **F32) / hidden ** 0.5).to(dtype)
        self.out = (torch.randn(heads * dim, hidden, **F32) / (heads * dim) ** 0.5).to(dtype)
        self.frequencies = L.DeviceRotary.Frequencies(dim)

    def project(self, x):
        rows = x @ self.qkv
        sizes = (self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim)
        return (part.unflatten(1, (-1, self.dim)) for part in rows.split(sizes, 1))

    def train_forward(self, x, lengths):
        """Causal attention over whole sequences laid end to end, without a cache."""
        q, k, v = self.project(x)
        positions = torch.cat([torch.arange(n, **I32) for n in lengths])
        q, k = Rotated.apply(q.contiguous(), k.contiguous(), positions, self.frequencies)
        rows, at = [], 0
        for n in lengths:
            qs = q[at:at + n].unflatten(1, (self.kv_heads, -1)).permute(1, 2, 0, 3)
            ks, vs = (t[at:at + n].permute(1, 0, 2)[:, None] for t in (k, v))
            logits = (qs.float() @ ks.float().transpose(-1, -2)) * self.dim ** -0.5
            ahead = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            share = torch.softmax(logits.masked_fill(ahead, float("-inf")), -1)
            rows.append((share @ vs.float()).permute(2, 0, 1, 3).reshape(n, -1))
            at += n
        return torch.cat(rows).to(x.dtype) @ self.out


class Cache:
    """The pages of one layer and the tables of the requests that share them."""

    def __init__(self, layer, requests, pages, block=16, width=16, budget=96):
        self.layer, self.n, self.block, self.budget = layer, requests, block, budget
        shape = (pages, block, layer.kv_heads, layer.dim)
        self.k, self.v = (torch.zeros(shape, dtype=layer.dtype, device="cuda") for _ in range(2))
        self.table = torch.full((requests, width), -1, **I32)
        self.free, self.used = torch.arange(pages, **I32), torch.zeros(1, **I32)
        self.lens, self.evicted = torch.zeros(requests, **I32), torch.zeros(requests, **I32)
        self.scores, self.positions = torch.zeros(pages * block, **F32), torch.zeros(pages * block, **I32)
        self.attention_temp = L.alloc_temp(L.DevicePagedAttention.GetTempStorageBytes(
            requests, layer.heads, layer.kv_heads, layer.dim, pages * block))
        self.moves = torch.zeros(requests, budget, 2, dtype=torch.int64, device="cuda")

    def step(self, x, new=None):
        """x: the step's tokens, request after request (one each unless `new` has their numbers).
        The layer's output for each request's last token."""
        n, tokens, layer = self.n, x.shape[0], self.layer
        temp = L.alloc_temp(L.DeviceBlockTable.GetTempStorageBytes(n, tokens))
        used, lens, starts = torch.zeros(1, **I32), torch.zeros(n, **I32), torch.zeros(n + 1, **I32)
        slots = torch.zeros(tokens, dtype=torch.int64, device="cuda")
        positions, requests = torch.zeros(tokens, **I32), torch.zeros(tokens, **I32)
        L.DeviceBlockTable().Extend(temp, self.lens, new, self.table, self.free, self.used, used, lens, starts, slots,
                                    positions, requests, n, self.block)
        self.lens, self.used = lens, used
        q, k, v = layer.project(x)
        # positions in the sequence: those in the cache, and what has been evicted before them
        L.DeviceRotary().Append(q, k, v, q, self.k, self.v, slots, positions, layer.frequencies, tokens,
                                d_token_request=requests, d_position_offset=self.evicted,
                                d_slot_positions=self.positions, d_slot_scores=self.scores)
        last = q[(starts[1:] - 1).long()]
        out = torch.empty_like(last)
        L.DevicePagedAttention().Decode(self.attention_temp, last, self.k, self.v, self.table, self.lens, out, n,
                                        d_scores=self.scores, d_scores_out=self.scores)
        return out.flatten(1) @ layer.out

    def evict(self):
        """Requests a page and more over the budget keep their first tokens, their last ones and the heaviest."""
        n = self.n
        lens, evicted = torch.zeros(n, **I32), torch.zeros(n, **I32)
        counts, used = torch.zeros(n, **I32), torch.zeros(1, **I32)
        d = L.DeviceCacheEviction()
        d.Plan(self.lens, self.table, self.scores, lens, counts, self.moves, n, self.block, self.budget,
               trigger=self.budget + self.block - 1, keep_first=4, keep_recent=16, d_positions=self.positions,
               d_evicted=self.evicted, d_evicted_out=evicted, d_free_blocks=self.free, d_free_used=self.used,
               d_free_used_out=used)
        # every layer's cache moves by the same plan; scores and positions once
        d.Move(self.moves, counts, self.k, self.v, n, d_scores=self.scores, d_positions=self.positions)
        self.lens, self.evicted, self.used = lens, evicted, used


def main(steps=120):
    torch.manual_seed(0)
    layer = Layer()
    hidden, requests = layer.qkv.shape[0], 6
    cache = Cache(layer, requests, pages=60)
    prompts = torch.tensor([40, 90, 7, 64, 1, 33], **I32)
    x = torch.randn(int(prompts.sum()), hidden, **F32).to(layer.dtype)
    y = cache.step(x, prompts)
    for _ in range(steps):
        y = cache.step(torch.tanh(y.float() + torch.randn(requests, hidden, **F32)).to(layer.dtype))
        cache.evict()
    total = (cache.lens + cache.evicted).tolist()
    print("tokens so far", total)
    print("in the cache ", cache.lens.tolist(), "in", int(cache.used), "pages")
    assert total == (prompts + steps).tolist() and y.isfinite().all()
    assert int(cache.lens.max()) < cache.budget + cache.block
    assert int(cache.used) == sum(-(-n // cache.block) for n in cache.lens.tolist())

    lengths = [50, 17, 33]
    x = torch.randn(sum(lengths), hidden, **F32).to(layer.dtype).requires_grad_(True)
    loss = layer.train_forward(x, lengths).float().square().mean()
    loss.backward()
    print("training loss %.4f, gradient norm %.4f" % (float(loss.detach()), float(x.grad.float().norm())))
    return cache, y


if __name__ == "__main__":
    main()
