"""A small network that predicts splats from a stream of posed views.

One token per 16 x 16 tile of a view (its pixels and the ray through its
middle) goes through blocks of a gated recurrence, windowed attention in which
the first view's first tokens stay visible, and a feed-forward layer, each behind
a residual norm; every token ends as a few Gaussians on its ray.  The whole
stream is trained at once through ``rasterize`` (``SplatPredictor.forward``);
afterwards views come one at a time, token after token, in constant memory
(``SplatPredictor.step``).

``python -m gaussian_splats_hip.sequence.predictor`` trains one on views of a
synthetic scene and streams the same views through it.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F
from torch import nn

from ..splats import GaussianSplat, PinholeCamera, SH_C0, rasterize
from ..training import l1_loss
from .attention import WindowCache, window_attention
from .norm import add_rms_norm
from .scan import gated_scan, gated_scan_step

TILE = 16


def view_tokens(image: torch.Tensor, camera: PinholeCamera) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens [tiles, 3 * 16 * 16 + 6] of an image [H, W, 3] whose sides are
    multiples of 16, and their rays [tiles, 6] (origin, direction)."""
    h, w = image.shape[0] // TILE, image.shape[1] // TILE
    pixels = image.reshape(h, TILE, w, TILE, 3).transpose(1, 2).reshape(h * w, -1)
    v, u = torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij")
    (fx, fy), (cx, cy) = camera.focal_length, camera.principal_point
    x = ((u + 0.5) * TILE - cx) / fx
    y = -((v + 0.5) * TILE - cy) / fy
    rotation = camera.rotation_matrix.cpu()
    direction = F.normalize(torch.stack((x, y, -torch.ones_like(x)), -1).reshape(-1, 3), dim=-1) @ rotation
    origin = camera.position.cpu().expand_as(direction)
    rays = torch.cat((origin, direction), -1).to(image)
    return torch.cat((pixels, rays), -1), rays


class Block(nn.Module):
    """Recurrence, attention and a feed-forward layer, each added to the
    float32 residual stream by the next one's norm."""

    def __init__(self, width: int, heads: int, kv_heads: int, window: int, sinks: int, dtype: torch.dtype):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.window, self.sinks = window, sinks
        self.norms = nn.Parameter(torch.ones(3, width))
        self.scan_in = nn.Linear(width, 2 * width, dtype=dtype)
        self.scan_out = nn.Linear(width, width, bias=False, dtype=dtype)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim, bias=False, dtype=dtype)
        self.attention_out = nn.Linear(width, width, bias=False, dtype=dtype)
        self.up = nn.Linear(width, 4 * width, dtype=dtype)
        self.down = nn.Linear(4 * width, width, dtype=dtype)
        # Gates that remember 3 to 3000 tokens, shorter and longer ones side by side.
        with torch.no_grad():
            self.scan_in.bias[width:] = torch.linspace(1.0, 8.0, width).to(dtype)

    def _qkv(self, y: torch.Tensor):
        q, k, v = self.qkv(y).split([self.heads * self.dim, self.kv_heads * self.dim,
                                     self.kv_heads * self.dim], -1)
        shape = y.shape[:-1]
        return (q.reshape(*shape, self.heads, self.dim), k.reshape(*shape, self.kv_heads, self.dim),
                v.reshape(*shape, self.kv_heads, self.dim))

    def forward(self, x: torch.Tensor, stream: torch.Tensor):
        """``x`` [batch, tokens, width], the last branch's output, and the
        stream it is to be added to; returns the same pair."""
        y, stream = add_rms_norm(x, stream, self.norms[0])
        value, gate = self.scan_in(y).chunk(2, -1)
        y, stream = add_rms_norm(self.scan_out(gated_scan(value, gate)[0]), stream, self.norms[1])
        out = window_attention(*self._qkv(y), self.window, self.sinks)
        y, stream = add_rms_norm(self.attention_out(out.flatten(-2)), stream, self.norms[2])
        return self.down(F.gelu(self.up(y))), stream

    def step(self, x: torch.Tensor, stream: torch.Tensor, state: torch.Tensor, cache: WindowCache):
        """One token of each stream: x and stream [batch, width]; ``state`` and
        ``cache`` move on by it."""
        y, stream = add_rms_norm(x, stream, self.norms[0])
        value, gate = self.scan_in(y).chunk(2, -1)
        mixed, _ = gated_scan_step(value, gate, state, state_out=state)
        y, stream = add_rms_norm(self.scan_out(mixed), stream, self.norms[1])
        out = cache.step(*self._qkv(y))
        y, stream = add_rms_norm(self.attention_out(out.flatten(-2)), stream, self.norms[2])
        return self.down(F.gelu(self.up(y))), stream


class SplatPredictor(nn.Module):
    def __init__(self, width: int = 256, heads: int = 4, kv_heads: int = 2, blocks: int = 2,
                 window: int = 512, sinks: int = 16, splats_per_token: int = 4,
                 depth: float = 3.0, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if width % heads or width // heads % 8:
            raise ValueError(f"width {width} does not give {heads} heads of a multiple of 8")
        self.depth, self.splats_per_token, self.width, self.dtype = depth, splats_per_token, width, dtype
        self.embed = nn.Linear(3 * TILE * TILE + 6, width, dtype=dtype)
        self.blocks = nn.ModuleList(
            Block(width, heads, kv_heads, window, sinks, dtype) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(width))
        # Per splat: depth, offset 3, rotation 4, log scale 3, opacity, colour 3.
        self.head = nn.Linear(width, 15 * splats_per_token, dtype=dtype)

    def _splats(self, y: torch.Tensor, rays: torch.Tensor) -> dict[str, torch.Tensor]:
        f = self.head(y).float().reshape(-1, self.splats_per_token, 15)
        depth, offset, rotation, scale, opacity, color = f.split([1, 3, 4, 3, 1, 3], -1)
        origin, direction = rays.reshape(-1, 1, 6).split(3, -1)
        unit = torch.tensor([1.0, 0.0, 0.0, 0.0], device=f.device)
        mean = origin + direction * self.depth * torch.exp(0.2 * depth) + 0.1 * offset
        return {"mean": mean.flatten(0, 1), "rotation": (rotation + unit).flatten(0, 1),
                "scale": (scale - 2.5).flatten(0, 1), "opacity": opacity.flatten(0, 1),
                "color": (color / SH_C0).reshape(-1, 1, 3)}

    def forward(self, tokens: torch.Tensor, rays: torch.Tensor) -> dict[str, torch.Tensor]:
        """Splat parameters of a stream's tokens [tokens, features] and rays
        [tokens, 6], for :func:`splats_of`."""
        x = self.embed(tokens.to(self.dtype))[None]
        stream = torch.zeros(x.shape, device=x.device)
        for block in self.blocks:
            x, stream = block(x, stream)
        return self._splats(add_rms_norm(x, stream, self.norm)[0], rays)

    def start(self, streams: int = 1) -> list[tuple[torch.Tensor, WindowCache]]:
        """States of ``streams`` running streams, one pair for each block."""
        device = self.norm.device
        return [(torch.zeros(streams, self.width, device=device),
                 WindowCache(streams, b.kv_heads, b.dim, b.window, b.sinks, self.dtype, device))
                for b in self.blocks]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, rays: torch.Tensor, states) -> dict[str, torch.Tensor]:
        """Splats of the next token of each stream (tokens [streams, features])."""
        x = self.embed(tokens.to(self.dtype))
        stream = torch.zeros(x.shape, device=x.device)
        for block, (state, cache) in zip(self.blocks, states):
            x, stream = block.step(x, stream, state, cache)
        return self._splats(add_rms_norm(x, stream, self.norm)[0], rays)


def splats_of(params: dict[str, torch.Tensor]) -> GaussianSplat:
    """A :class:`GaussianSplat` that keeps the parameters' graph, so that a
    loss on its image reaches the network."""
    splats = GaussianSplat(0, 0)
    for name, value in params.items():
        del splats._parameters[name]
        setattr(splats, name, value)
    return splats


def _views(device: torch.device, count: int, size: int, seed: int):
    """Images of a seeded scene from cameras around it."""
    g = torch.Generator().manual_seed(seed)
    n = 2000
    scene = GaussianSplat.from_tensors(
        torch.rand(n, 3, generator=g) * 1.6 - 0.8, torch.randn(n, 4, generator=g),
        torch.randn(n, 3, generator=g) * 0.3 - 2.8, torch.randn(n, 1, generator=g) + 1,
        torch.randn(n, 1, 3, generator=g) * 0.8).to(device)
    angles = torch.arange(count) * (2 * torch.pi / (4 * count))
    cameras = [PinholeCamera.look_at((3 * float(a.sin()), 0.5, -3 * float(a.cos())), image_size=(size, size),
                                     focal_length=(float(size), float(size)),
                                     principal_point=(size / 2, size / 2)) for a in angles]
    with torch.no_grad():
        return cameras, [rasterize(scene, c, tile_size=TILE).clamp(0, 1) for c in cameras]


def train(steps: int = 60, views: int = 4, size: int = 128, seed: int = 0, device: str = "cuda",
          log=print) -> tuple[SplatPredictor, torch.Tensor, torch.Tensor, list[float]]:
    """Fits a predictor to the views of one synthetic scene; returns it with the
    stream's tokens, their rays and the losses."""
    torch.manual_seed(seed)
    device = torch.device(device)
    cameras, images = _views(device, views, size, seed)
    pairs = [view_tokens(i, c) for i, c in zip(images, cameras)]
    tokens, rays = torch.cat([t for t, _ in pairs]), torch.cat([r for _, r in pairs])
    # A window of one view and a half.
    model = SplatPredictor(window=tokens.shape[0] * 3 // (2 * views)).to(device)
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    losses = []
    for step in range(steps):
        splats = splats_of(model(tokens, rays))
        loss = sum(l1_loss(rasterize(splats, c, tile_size=TILE), i, clamp=True)
                   for c, i in zip(cameras, images)) / views
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step}: l1 {losses[-1]:.4f}")
    return model, tokens, rays, losses


@torch.no_grad()
def stream(model: SplatPredictor, tokens: torch.Tensor, rays: torch.Tensor) -> dict[str, torch.Tensor]:
    """The same splats as ``model(tokens, rays)``, one token at a time."""
    states = model.start()
    parts = [model.step(tokens[t:t + 1], rays[t:t + 1], states) for t in range(tokens.shape[0])]
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--views", type=int, default=4)
    parser.add_argument("--size", type=int, default=128, help="image side, a multiple of 16")
    args = parser.parse_args()
    model, tokens, rays, _ = train(args.steps, args.views, args.size)
    with torch.no_grad():
        whole = model(tokens, rays)
    streamed = stream(model, tokens, rays)
    off = max(float((whole[k] - streamed[k]).abs().max()) for k in whole)
    print(f"{tokens.shape[0]} tokens streamed one at a time: {streamed['mean'].shape[0]} splats, "
          f"largest difference from the whole stream's {off:.3f}")


if __name__ == "__main__":
    main()
