"""Prompted points against a volume that is held on the GPU in 8 bits, with 4-bit weights.

The volume's tokens pass a transformer block once (examples/volume_tokens.py has the blocks); what stays of them
are the keys and values of its last layer, quantised as they are written.  A batch of points is then one token each:

    norm -> queries, keys, values (4-bit weights) -> rotary positions
         -> held behind the volume's tokens -> attention over all that is held
         -> projection (4 bits) -> residual sum and norm
         -> gated feed-forward (4 bits, gate and product in one) -> narrowing product (4 bits) -> residual sum and norm

so that every point sees the volume and the points before it.  Run it on a GPU host, from the repository's root:

    PYTHONPATH=nnunet-mlx_amd python examples/held_volume.py --size 128 --cube 8 --points 4
"""

from __future__ import annotations

import argparse

import torch

from nnunet_mlx.model import tokens


class PointBlock:
    """One block with random weights, packed to 4 bits."""

    def __init__(self, *, heads: int = 5, kv_heads: int = 5, head_dim: int = 64, hidden: int = 1280, group: int = 64,
                 dtype: torch.dtype = torch.bfloat16, seed: int = 0):
        gen = torch.Generator().manual_seed(seed)
        width = heads * head_dim

        def packed(outputs: int, inputs: int) -> tokens.PackedWeight:
            return tokens.pack_weight((torch.randn(outputs, inputs, generator=gen) * inputs**-0.5).to(dtype).cuda(), group)

        def weight() -> tuple[torch.Tensor, None]:
            return (1 + 0.1 * torch.randn(width, generator=gen)).cuda(), None

        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        self.plan = tokens.rotary_plan(head_dim // 6 * 6, axes=3, base=100.0)
        self.qkv, self.out = packed(width + 2 * kv_heads * head_dim, width), packed(width, width)
        self.gate, self.up, self.down = packed(hidden, width), packed(hidden, width), packed(width, hidden)
        self.pre, self.mlp_pre, self.next_pre = weight(), weight(), weight()

    def project(self, y: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Rotated queries and keys, and values, of normed tokens (batch, tokens, width)."""
        qkv = tokens.packed_linear(y, self.qkv).unflatten(-1, (-1, self.head_dim))
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 2)
        q, k = tokens.rotate(q, k, positions, self.plan)
        return q, k, v

    def hold(self, x: torch.Tensor, positions: torch.Tensor, room: int) -> tokens.HeldTokens:
        """The keys and values of a volume's tokens (batch, tokens, width), with room for more tokens behind them."""
        _, y = tokens.residual_norm(x, None, kind="rms", pre=self.pre)
        _, k, v = self.project(y, positions)
        held = tokens.held_tokens(x.shape[0], x.shape[1] + room, self.kv_heads, self.head_dim)
        return tokens.hold_tokens(held, k, v)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, held: tokens.HeldTokens,
                 lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Points (batch, points, width) after the block, and their next norm.  They are held behind each item's
        ``lengths`` int32 (batch,) slots, which then count them too."""
        residual, y = tokens.residual_norm(x, None, kind="rms", pre=self.pre)
        q, k, v = self.project(y, positions)
        tokens.hold_tokens(held, k, v, start=lengths)
        start = lengths.clone()
        lengths += x.shape[1]
        mixed = tokens.held_attention(q, held, lengths, causal=True, start=start)
        residual, y = tokens.residual_norm(tokens.packed_linear(mixed.flatten(2), self.out), residual, kind="rms",
                                           pre=self.mlp_pre)
        hidden = tokens.packed_linear(y, self.up, gate=self.gate, gate_activation="silu")
        return tokens.residual_norm(tokens.packed_linear(hidden, self.down), residual, kind="rms", pre=self.next_pre)


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--size", type=int, default=128, help="side of the volume, a multiple of the cube's")
    parser.add_argument("--cube", type=int, default=8)
    parser.add_argument("--points", type=int, default=4)
    args = parser.parse_args()
    side = args.size // args.cube
    block = PointBlock()
    gen = torch.Generator().manual_seed(1)
    width = block.heads * block.head_dim
    axes = [torch.arange(side, dtype=torch.int32)] * 3
    positions = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3).cuda()
    volume = torch.randn(1, side**3, width, generator=gen).to(block.dtype).cuda()
    held = block.hold(volume, positions, room=64 * args.points)
    lengths = torch.full((1,), side**3, dtype=torch.int32, device="cuda")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    answers = []
    for step in range(12):
        points = torch.randn(1, args.points, width, generator=gen).to(block.dtype).cuda()
        at = torch.randint(0, side, (args.points, 3), generator=gen, dtype=torch.int32).cuda()
        if step == 2:
            start.record()
        answers.append(block(points, at, held, lengths)[1])
    end.record()
    torch.cuda.synchronize()
    held_bytes = sum(t.numel() * t.element_size() for t in held)
    print(f"{side**3} tokens held in {held_bytes / 1e6:.1f} MB; {args.points} points a step: "
          f"{start.elapsed_time(end) / 10:.3f} ms; the last answer has norm {float(answers[-1].float().norm()):.3f}")


if __name__ == "__main__":
    main()
