"""One attention layer that trains on whole rows and answers a token at a time.

    python examples/streaming_layer.py [--steps 20] [--prompt 700] [--new 64]

Training uses fa.window_attention (a sliding window and a few first tokens, with gradients); serving
appends the prompt and then every new token to an e4m3 paged cache with fa.append_kv, which turns
queries and keys by their positions on the way, and attends over it with fa.forward_cached. Both see
the same keys, so the layer's answers to the same tokens agree up to e4m3's rounding, which the
example prints. The decoding step is captured in a CUDA graph: lengths live on the device.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "flash-attention-from-scratch_b200"))

import fa  # noqa: E402


class StreamingAttention(torch.nn.Module):
    """Grouped-head attention over a window and the first tokens, with rotated positions."""

    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, window: int, sinks: int, rows: int, device) -> None:
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.window, self.sinks = heads, kv_heads, head_dim, window, sinks
        make = lambda i, o: torch.nn.Linear(i, o, bias=False, device=device, dtype=torch.bfloat16)  # noqa: E731
        self.qkv = make(width, (heads + 2 * kv_heads) * head_dim)
        self.out = make(heads * head_dim, width)
        turn = torch.arange(rows, device=device)[:, None] * 10000.0 ** (
            -torch.arange(head_dim // 2, device=device) * 2 / head_dim)
        self.register_buffer("cos", turn.cos().contiguous())
        self.register_buffer("sin", turn.sin().contiguous())

    def split(self, x: torch.Tensor):
        """q, k, v as [B, H, N, D] views of one projection."""
        b, n, _ = x.shape
        y = self.qkv(x).view(b, n, self.heads + 2 * self.kv_heads, self.head_dim)
        return (t.transpose(1, 2) for t in y.split([self.heads, self.kv_heads, self.kv_heads], 2))

    def turned(self, x: torch.Tensor) -> torch.Tensor:
        """Rotation of whole rows in torch, differentiable (serving rotates in append_kv)."""
        a, b = x.float().chunk(2, -1)
        c, s = self.cos[: x.shape[2]], self.sin[: x.shape[2]]
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)

    def merge(self, o: torch.Tensor) -> torch.Tensor:
        b, _, n, _ = o.shape
        return self.out(o.transpose(1, 2).reshape(b, n, -1))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q, k, v = self.split(x)
        return self.merge(fa.window_attention(self.turned(q), self.turned(k), v, self.window, sinks=self.sinks))

    @torch.no_grad()
    def serve(self, x: torch.Tensor, cache, table: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        """The layer's output for the newest tokens x [B, T, width]; lengths count them already."""
        q, k, v = self.split(x)
        q = fa.append_kv(cache, k, v, table, lengths, cos=self.cos, sin=self.sin, q=q)
        return self.merge(fa.forward_cached(q, cache, table, lengths, window=self.window, sinks=self.sinks))


def main(argv: list[str] | None = None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20, help="training steps")
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--new", type=int, default=64, help="tokens answered after the prompt")
    ap.add_argument("--batch", type=int, default=2)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    device = torch.device("cuda", torch.cuda.current_device())
    width, rows, page = 256, a.prompt + a.new, 64
    layer = StreamingAttention(width, 8, 2, 64, window=256, sinks=4, rows=rows, device=device)

    # Train: recall the token two places back.
    tokens = torch.randn(a.batch, rows, width, device=device, dtype=torch.bfloat16)
    target = tokens.roll(2, 1)
    optimiser = torch.optim.AdamW(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(a.steps):
        optimiser.zero_grad(set_to_none=True)
        loss = (layer(tokens) - target)[:, 2:].float().square().mean()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    losses = [float(x) for x in losses]

    # Serve the same tokens: the prompt at once, then one at a time from a graph.
    per = -(-rows // page)
    cache = fa.PagedKVCache.empty(a.batch * per, page, layer.kv_heads, layer.head_dim, device=device)
    table = torch.randperm(a.batch * per, device=device).to(torch.int32).view(a.batch, per)
    lengths = torch.full((a.batch,), a.prompt, dtype=torch.int32, device=device)
    served = [layer.serve(tokens[:, : a.prompt], cache, table, lengths)]
    if a.new > 0:
        token = tokens[:, a.prompt : a.prompt + 1].clone()

        def step() -> torch.Tensor:
            lengths.add_(1)
            return layer.serve(token, cache, table, lengths)

        served.append(step())  # the first one outside the graph warms up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            answer = step()
        for i in range(a.prompt + 1, rows):
            token.copy_(tokens[:, i : i + 1])
            graph.replay()
            served.append(answer.clone())
    with torch.no_grad():
        whole = layer(tokens)
    off = (torch.cat(served, 1).float() - whole.float()).norm() / whole.float().norm()
    result = {"first_loss": losses[0] if losses else None, "last_loss": losses[-1] if losses else None,
              "served_against_whole": float(off), "status": fa._C.device_status(device.index)}
    print(result)
    return result


if __name__ == "__main__":
    main()
