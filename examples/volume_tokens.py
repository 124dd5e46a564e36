"""Transformer blocks over the tokens of a volume, with the token operators together.

A volume is cut into cubes, one token each.  A block is

    norm -> queries, keys, values -> rotary positions of the cube's three coordinates
         -> attention over the blocks of tokens that each token selects, background cubes masked
         -> projection -> norm of the branch, scale, residual sum and the norm of the next half
         -> two-layer perceptron -> the same again

and a last step answers a single prompted point against the held keys of the volume.  The plain
matrix products are torch's.  Run it on a GPU host, from the repository's root:

    PYTHONPATH=nnunet-mlx_amd python examples/volume_tokens.py --size 128 --cube 8
"""

from __future__ import annotations

import argparse
from typing import NamedTuple

import torch

from nnunet_mlx.model import tokens


class Cubes(NamedTuple):
    """Flattened cubes (1, tokens, cube^3), their coordinates (tokens, 3) and which hold anything."""

    voxels: torch.Tensor
    positions: torch.Tensor
    foreground: torch.Tensor


def cut(volume: torch.Tensor, cube: int) -> Cubes:
    """Cubes of a (Z, Y, X) volume whose sides are multiples of ``cube``."""
    z, y, x = (n // cube for n in volume.shape)
    voxels = volume.reshape(z, cube, y, cube, x, cube).permute(0, 2, 4, 1, 3, 5).reshape(1, z * y * x, cube**3)
    axes = [torch.arange(n, dtype=torch.int32, device=volume.device) for n in (z, y, x)]
    positions = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3).contiguous()
    return Cubes(voxels, positions, (voxels != 0).any(-1).contiguous())


class VolumeTokens:
    """A few such blocks with random weights."""

    def __init__(self, cube: int = 8, *, heads: int = 5, head_dim: int = 64, depth: int = 2, block: int = 64,
                 keep: int = 16, dtype: torch.dtype = torch.bfloat16, seed: int = 0):
        gen = torch.Generator().manual_seed(seed)
        width = heads * head_dim

        def matrix(rows: int, columns: int) -> torch.Tensor:
            return (torch.randn(rows, columns, generator=gen) * rows**-0.5).to(dtype).cuda()

        def affine() -> tuple[torch.Tensor, torch.Tensor]:
            return ((1 + 0.1 * torch.randn(width, generator=gen)).cuda(), (0.1 * torch.randn(width, generator=gen)).cuda())

        self.heads, self.head_dim, self.block, self.keep, self.dtype = heads, head_dim, block, keep, dtype
        # three coordinates turn 20 elements of a head each, as far as the head goes
        self.plan = tokens.rotary_plan(head_dim // 6 * 6, axes=3, base=100.0)
        self.embed, self.first_norm = matrix(cube**3, width), affine()
        self.layers = [{"qkv": matrix(width, 3 * width), "out": matrix(width, width), "up": matrix(width, 4 * width),
                        "down": matrix(4 * width, width), "post": affine(), "mlp_pre": affine(),
                        "mlp_post": affine(), "next_pre": affine(),
                        "scale": (0.2 + 0.05 * torch.randn(width, generator=gen)).cuda()} for _ in range(depth)]

    def __call__(self, cubes: Cubes) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """Tokens (1, tokens, width) after the blocks' last norm, the kept blocks of the last layer, and its
        rotated keys and its values."""
        residual, y = tokens.residual_norm(cubes.voxels.to(self.dtype) @ self.embed, None, pre=self.first_norm)
        for layer in self.layers:
            qkv = (y @ layer["qkv"]).unflatten(-1, (3 * self.heads, self.head_dim))
            q, k, v = qkv.split(self.heads, 2)
            q, k = tokens.rotate(q, k, cubes.positions, self.plan)
            mixed, kept = tokens.sparse_attention(q, k, v, self.block, self.keep, key_mask=cubes.foreground)
            residual, y = tokens.residual_norm(mixed.flatten(2) @ layer["out"], residual, post=layer["post"],
                                               scale=layer["scale"], pre=layer["mlp_pre"])
            branch = torch.nn.functional.gelu(y @ layer["up"]) @ layer["down"]
            residual, y = tokens.residual_norm(branch, residual, post=layer["mlp_post"], scale=layer["scale"],
                                               pre=layer["next_pre"])
        return y, kept, k, v

    def point(self, query: torch.Tensor, at: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
              summary: tokens.BlockSummary, foreground: torch.Tensor) -> torch.Tensor:
        """One point's query (1, 1, heads, head_dim) at coordinates (1, 3) against held keys, whose
        summary is held too."""
        query, _ = tokens.rotate(query, None, at, self.plan)
        mixed, _ = tokens.sparse_attention(query, keys, values, self.block, self.keep, summary=summary, local=0,
                                           key_mask=foreground)
        return mixed


def phantom(size: int, seed: int = 0) -> torch.Tensor:
    """A (size, size, size) ball of smooth texture in an empty background."""
    gen = torch.Generator().manual_seed(seed)
    coarse = torch.randn(1, 1, 8, 8, 8, generator=gen)
    texture = torch.nn.functional.interpolate(coarse, size=(size,) * 3, mode="trilinear", align_corners=False)[0, 0]
    axis = torch.linspace(-1, 1, size)
    inside = axis[:, None, None] ** 2 + axis[None, :, None] ** 2 + axis[None, None, :] ** 2 < 0.8
    return (texture * inside).cuda()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--size", type=int, default=128, help="side of the volume, a multiple of the cube's")
    parser.add_argument("--cube", type=int, default=8)
    parser.add_argument("--keep", type=int, default=16)
    args = parser.parse_args()
    net = VolumeTokens(args.cube, keep=args.keep)
    cubes = cut(phantom(args.size), args.cube)
    y, kept, k, v = net(cubes)
    summary = tokens.summarize_blocks(k, net.block, key_mask=cubes.foreground)
    query = torch.randn(1, 1, net.heads, net.head_dim, generator=torch.Generator().manual_seed(1)).to(net.dtype).cuda()
    middle = torch.full((1, 3), args.size // args.cube // 2, dtype=torch.int32, device="cuda")
    answer = net.point(query, middle, k, v, summary, cubes.foreground)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(10):
        net(cubes)
    end.record()
    torch.cuda.synchronize()
    print(f"{y.shape[1]} tokens ({int(cubes.foreground.sum())} of them foreground), {len(net.layers)} blocks: "
          f"{start.elapsed_time(end) / 10:.3f} ms; a token keeps {int((kept >= 0).sum(-1).max())} of "
          f"{summary.scales.shape[2]} blocks; a point's answer has norm {float(answer.float().norm()):.3f}")


if __name__ == "__main__":
    main()
