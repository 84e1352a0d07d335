"""One differential attention layer, trained for a few steps and then served from the 4-bit cache.

    python examples/differential_layer.py

Training runs ``differential_softmax_attention`` with shared key / value heads
and lambda learned as exp(a.b) - exp(c.d) + init per head.  Serving packs
prompts of uneven length: ``plan_pages`` hands out pages and slots,
``cache4_append`` writes the prompt's keys and values, and each decode step is
plan, append, ``cache4_softmax_attention``, captured once in a CUDA graph and
replayed.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import tda_b200  # noqa: E402


class DifferentialLayer(torch.nn.Module):
    def __init__(self, width=256, heads=8, kv_heads=2, head_dim=64, lambda_init=0.3, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.lambda_init = heads, kv_heads, head_dim, lambda_init
        kw = dict(bias=False, device=device, dtype=dtype)
        self.q = torch.nn.Linear(width, 2 * heads * head_dim, **kw)
        self.kv = torch.nn.Linear(width, 3 * kv_heads * head_dim, **kw)
        self.out = torch.nn.Linear(heads * head_dim, width, **kw)
        self.lam = torch.nn.Parameter(0.1 * torch.randn(4, heads, head_dim, device=device))

    def weight(self):
        a, b, c, d = self.lam
        return (torch.exp((a * b).sum(-1)) - torch.exp((c * d).sum(-1)) + self.lambda_init).reshape(1, -1, 1, 1)

    def project(self, x):
        """q1, q2 (..., heads, D) and k1, k2, v (..., kv heads, D) of x (..., width): views of two products."""
        q = self.q(x).unflatten(-1, (2, self.heads, self.head_dim))
        kv = self.kv(x).unflatten(-1, (3, self.kv_heads, self.head_dim))
        return q[..., 0, :, :], q[..., 1, :, :], kv[..., 0, :, :], kv[..., 1, :, :], kv[..., 2, :, :]

    def forward(self, x, key_lengths=None):
        heads_first = [t.transpose(1, 2) for t in self.project(x)]  # read in place, no copies
        o = tda_b200.differential_softmax_attention(*heads_first, self.weight(), key_lengths=key_lengths)
        return self.out(o.transpose(1, 2).flatten(2))


def train(layer, steps=20, batch=4, length=200, seed=0):
    """Fit the layer to a running mean of its inputs; the losses of the steps."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = layer.q.in_features
    opt = torch.optim.Adam(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        x = torch.randn(batch, length, width, generator=gen, device="cuda").to(layer.q.weight.dtype)
        target = x.float().cumsum(1) / torch.arange(1, length + 1, device="cuda")[:, None]
        loss = (layer(x).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


class Server:
    """A batch of requests over one layer's 4-bit cache."""

    def __init__(self, layer, requests, longest, page_size=32):
        self.layer, self.page = layer, page_size
        width = -(-longest // page_size)
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.cache = tda_b200.Cache4(requests * width, page_size, layer.kv_heads, layer.head_dim)
        self.table = ints(requests, width) - 1
        self.free = torch.arange(requests * width, dtype=torch.int32, device="cuda")
        self.head, self.lengths = ints(1), ints(requests)
        self.ones = ints(requests) + 1
        self.graph = None

    @torch.no_grad()
    def prefill(self, x, prompt_lengths):
        """x (requests, longest prompt, width), padded; returns the layer's output for it."""
        new = prompt_lengths.to(torch.int32)
        y = self.layer(x, key_lengths=new)
        plan = tda_b200.plan_pages(self.lengths, new, self.table, self.free, self.head, self.page, x.shape[0] * x.shape[1])
        # packed rows in the plan's order; rows past the last token point at a token and have no slot
        rows = x[plan.requests.clamp(min=0).long(), plan.positions.clamp(min=0).long()]
        _, _, k1, k2, v = self.layer.project(rows)
        tda_b200.cache4_append(self.cache, k1, k2, v, plan.slots)
        self.lengths.copy_(plan.lengths)
        self.head.copy_(plan.free_head)
        return y

    @torch.no_grad()
    def _step(self):
        q1, q2, k1, k2, v = self.layer.project(self.x)
        plan = tda_b200.plan_pages(self.lengths, self.ones, self.table, self.free, self.head, self.page, self.x.shape[0])
        tda_b200.cache4_append(self.cache, k1, k2, v, plan.slots)
        o = tda_b200.cache4_softmax_attention(q1, q2, self.cache, self.table, plan.lengths, self.layer.weight())
        self.lengths.copy_(plan.lengths)
        self.head.copy_(plan.free_head)
        return self.layer.out(o.flatten(1))

    def decode(self, x):
        """One token a request, x (requests, width): its output.  The first call captures the step."""
        if self.graph is None:
            self.x = x.clone()
            held = [t.clone() for t in (self.lengths, self.head, self.table)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self._step()
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.y = self._step()
            for t, h in zip((self.lengths, self.head, self.table), held):  # the warm-up's token is written again
                t.copy_(h)
        self.x.copy_(x)
        self.graph.replay()
        return self.y


def main(steps=20, decode_steps=40, seed=0):
    torch.manual_seed(seed)
    layer = DifferentialLayer()
    losses = train(layer, steps, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    prompts = torch.tensor([70, 1, 33, 128], device="cuda")
    total = int(prompts.max()) + decode_steps
    x = torch.randn(4, total, layer.q.in_features, generator=gen, device="cuda").to(layer.q.weight.dtype)
    server = Server(layer, 4, total)
    server.prefill(x[:, :int(prompts.max())], prompts)
    rows = torch.arange(4, device="cuda")
    served, exact = [], []
    with torch.no_grad():
        for n in range(decode_steps):
            at = prompts + n
            served.append(server.decode(x[rows, at]).clone())
            exact.append(torch.stack([layer(x[b:b + 1, :int(at[b]) + 1])[0, -1] for b in range(4)]))
    served, exact = torch.stack(served).float(), torch.stack(exact).float()
    drift = float((served - exact).norm() / exact.norm())
    return losses, drift, server.lengths.tolist(), (prompts + decode_steps).tolist()


if __name__ == "__main__":
    losses, drift, lengths, _ = main()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; decode from 4 bits is {100 * drift:.1f}% off the bf16 layer; "
          f"tokens held {lengths}")
