"""A small network that predicts splats from a stream of posed views.

One token per 16 x 16 tile of a view (its pixels and the ray through its
middle) goes through blocks of a recurrence, windowed attention in which
the first view's first tokens stay visible, and a feed-forward layer, each behind
a residual norm; every token ends as a few Gaussians on its ray.  The recurrence
is a gated mean of each channel, or the gated delta rule, which writes to a matrix
per head what its keys do not read there yet.  The whole stream is trained at once
through ``rasterize`` (``SplatPredictor.forward``); afterwards views come one at a
time, token after token, in constant memory (``SplatPredictor.step``), with the
attention's cache in the network's type or in 4 bits.

``python -m gaussian_splats_hip.sequence.predictor`` trains one on views of a
synthetic scene and streams the same views through it.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F
from torch import nn

from ..splats import GaussianSplat, PinholeCamera, SH_C0, rasterize
from ..training import clip_grad_norm, l1_loss
from .attention import WindowCache, window_attention
from .cache_quant import QuantWindowCache
from .delta import delta_scan, delta_scan_step
from .norm import add_rms_norm
from .scan import gated_scan, gated_scan_step

TILE = 16
MIXERS = ("gated", "delta")


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

    def __init__(self, width: int, heads: int, kv_heads: int, window: int, sinks: int, dtype: torch.dtype,
                 mixer: str = "gated"):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.window, self.sinks, self.mixer = window, sinks, mixer
        self.norms = nn.Parameter(torch.ones(3, width))
        # Value and gate of each channel; or query and key of each key head, value,
        # gate and writing strength of each head.
        keys = kv_heads * self.dim
        self.scan_parts = [width, width] if mixer == "gated" else [keys, keys, width, heads, heads]
        self.scan_in = nn.Linear(width, sum(self.scan_parts), dtype=dtype)
        self.scan_out = nn.Linear(width, width, bias=False, dtype=dtype)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim, bias=False, dtype=dtype)
        self.attention_out = nn.Linear(width, width, bias=False, dtype=dtype)
        self.up = nn.Linear(width, 4 * width, dtype=dtype)
        self.down = nn.Linear(4 * width, width, dtype=dtype)
        # Gates that remember 3 to 3000 tokens, shorter and longer ones side by side.
        with torch.no_grad():
            gate = self.scan_in.bias.split(self.scan_parts)[1 if mixer == "gated" else 3]
            gate.copy_(torch.linspace(1.0, 8.0, gate.numel()))

    def _qkv(self, y: torch.Tensor):
        q, k, v = self.qkv(y).split([self.heads * self.dim, self.kv_heads * self.dim,
                                     self.kv_heads * self.dim], -1)
        shape = y.shape[:-1]
        return (q.reshape(*shape, self.heads, self.dim), k.reshape(*shape, self.kv_heads, self.dim),
                v.reshape(*shape, self.kv_heads, self.dim))

    def _delta(self, y: torch.Tensor):
        """Queries and keys of length one, values, gates and writing strengths."""
        q, k, v, gate, beta = self.scan_in(y).split(self.scan_parts, -1)
        q, k = (F.normalize(t.unflatten(-1, (self.kv_heads, self.dim)).float(), dim=-1).to(y.dtype)
                for t in (q, k))
        return q, k, v.unflatten(-1, (self.heads, self.dim)), gate, beta

    def _mix(self, y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        if self.mixer == "gated":
            return gated_scan(*self.scan_in(y).chunk(2, -1))
        out, last = delta_scan(*self._delta(y), scale=1.0)
        return out.flatten(-2), last

    def _mix_step(self, y: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        if self.mixer == "gated":
            return gated_scan_step(*self.scan_in(y).chunk(2, -1), state, state_out=state)[0]
        return delta_scan_step(*self._delta(y), state, scale=1.0, state_out=state)[0].flatten(-2)

    def start(self, streams: int, cache_bits: int):
        """State and cache of streams without a token."""
        device = self.norms.device
        shape = (self.heads * self.dim,) if self.mixer == "gated" else (self.heads, self.dim, self.dim)
        sizes = (streams, self.kv_heads, self.dim, self.window, self.sinks)
        return (torch.zeros(streams, *shape, device=device),
                QuantWindowCache(*sizes, device=device) if cache_bits == 4
                else WindowCache(*sizes, self.up.weight.dtype, device))

    def forward(self, x: torch.Tensor, stream: torch.Tensor, state: torch.Tensor | None = None,
                cache: WindowCache | QuantWindowCache | None = None):
        """``x`` [batch, tokens, width], the last branch's output, and the
        stream it is to be added to; returns the same pair.  ``state`` and ``cache``,
        where given, are left as they stand behind the last token."""
        y, stream = add_rms_norm(x, stream, self.norms[0])
        mixed, last = self._mix(y)
        y, stream = add_rms_norm(self.scan_out(mixed), stream, self.norms[1])
        q, k, v = self._qkv(y)
        if cache is not None:
            # Both fit before either is written: copy_ alone would spread one sequence's
            # state over those of several streams.
            if state.shape != last.shape:
                raise ValueError(f"state {tuple(state.shape)} is not {list(last.shape)}, that of the tokens")
            cache.fill(k, v)
            state.copy_(last)
        out = window_attention(q, k, v, self.window, self.sinks)
        y, stream = add_rms_norm(self.attention_out(out.flatten(-2)), stream, self.norms[2])
        return self.down(F.gelu(self.up(y))), stream

    def step(self, x: torch.Tensor, stream: torch.Tensor, state: torch.Tensor,
             cache: WindowCache | QuantWindowCache):
        """One token of each stream: x and stream [batch, width]; ``state`` and
        ``cache`` move on by it."""
        y, stream = add_rms_norm(x, stream, self.norms[0])
        y, stream = add_rms_norm(self.scan_out(self._mix_step(y, state)), stream, self.norms[1])
        out = cache.step(*self._qkv(y))
        y, stream = add_rms_norm(self.attention_out(out.flatten(-2)), stream, self.norms[2])
        return self.down(F.gelu(self.up(y))), stream


class SplatPredictor(nn.Module):
    def __init__(self, width: int = 256, heads: int = 4, kv_heads: int = 2, blocks: int = 2,
                 window: int = 512, sinks: int = 16, splats_per_token: int = 4,
                 depth: float = 3.0, dtype: torch.dtype = torch.bfloat16, mixer: str = "gated"):
        super().__init__()
        if width % heads or width // heads % 8:
            raise ValueError(f"width {width} does not give {heads} heads of a multiple of 8")
        if mixer not in MIXERS:
            raise ValueError(f"mixer must be one of {MIXERS}, got {mixer!r}")
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
        self.depth, self.splats_per_token, self.width, self.dtype = depth, splats_per_token, width, dtype
        self.embed = nn.Linear(3 * TILE * TILE + 6, width, dtype=dtype)
        self.blocks = nn.ModuleList(
            Block(width, heads, kv_heads, window, sinks, dtype, mixer) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(width))
        # Per splat: depth, offset 3, rotation 4, log scale 3, opacity, colour 3.
        self.head = nn.Linear(width, 15 * splats_per_token, dtype=dtype)

    def _splats(self, y: torch.Tensor, rays: torch.Tensor) -> dict[str, torch.Tensor]:
        f = self.head(y).float().reshape(-1, self.splats_per_token, 15)
        depth, offset, rotation, scale, opacity, color = f.split([1, 3, 4, 3, 1, 3], -1)
        origin, direction = rays.reshape(-1, 1, 6).split(3, -1)
        unit = torch.eye(1, 4, device=f.device)
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

    def start(self, streams: int = 1, cache_bits: int = 16) -> list[tuple]:
        """States of ``streams`` running streams, a pair for each block: the
        recurrence's and the attention's cache, in the network's type or, with
        ``cache_bits`` 4, as a :class:`QuantWindowCache` (heads of a multiple of 32)."""
        if cache_bits not in (4, 16):
            raise ValueError(f"cache_bits must be 4 or 16 (the network's type), got {cache_bits}")
        return [b.start(streams, cache_bits) for b in self.blocks]

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, rays: torch.Tensor, states) -> dict[str, torch.Tensor]:
        """:meth:`forward` of the first tokens of one stream, whose ``states``
        (``start()``) then stand behind them for :meth:`step`."""
        x = self.embed(tokens.to(self.dtype))[None]
        stream = torch.zeros(x.shape, device=x.device)
        for block, (state, cache) in zip(self.blocks, states):
            x, stream = block(x, stream, state, cache)
        return self._splats(add_rms_norm(x, stream, self.norm)[0], rays)

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
          log=print, mixer: str = "gated", max_norm: float | None = None) -> tuple[SplatPredictor, torch.Tensor, torch.Tensor, list[float]]:
    """Fits a predictor to the views of one synthetic scene; returns it with the
    stream's tokens, their rays and the losses.  ``max_norm`` limits the gradients'
    norm in every step."""
    torch.manual_seed(seed)
    device = torch.device(device)
    cameras, images = _views(device, views, size, seed)
    pairs = [view_tokens(i, c) for i, c in zip(images, cameras)]
    tokens, rays = torch.cat([t for t, _ in pairs]), torch.cat([r for _, r in pairs])
    # A window of one view and a half.
    model = SplatPredictor(window=tokens.shape[0] * 3 // (2 * views), mixer=mixer).to(device)
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    losses = []
    for step in range(steps):
        splats = splats_of(model(tokens, rays))
        loss = sum(l1_loss(rasterize(splats, c, tile_size=TILE), i, clamp=True)
                   for c, i in zip(cameras, images)) / views
        optimizer.zero_grad()
        loss.backward()
        if max_norm is not None:
            clip_grad_norm(model.parameters(), max_norm)
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step}: l1 {losses[-1]:.4f}")
    return model, tokens, rays, losses


@torch.no_grad()
def stream(model: SplatPredictor, tokens: torch.Tensor, rays: torch.Tensor, cache_bits: int = 16,
           first: int = 0) -> dict[str, torch.Tensor]:
    """The same splats as ``model(tokens, rays)``, one token at a time behind the
    ``first`` ones, which are taken at once; with ``cache_bits`` 4 up to the cache's
    rounding."""
    states = model.start(cache_bits=cache_bits)
    parts = [model.prefill(tokens[:first], rays[:first], states)] if first else []
    parts += [model.step(tokens[t:t + 1], rays[t:t + 1], states) for t in range(first, tokens.shape[0])]
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--views", type=int, default=4)
    parser.add_argument("--size", type=int, default=128, help="image side, a multiple of 16")
    parser.add_argument("--mixer", choices=MIXERS, default="gated", help="the blocks' recurrence")
    parser.add_argument("--max-norm", type=float, help="limit of the gradients' norm (default: none)")
    parser.add_argument("--cache-bits", type=int, choices=(4, 16), default=16,
                        help="the streams' cache: in 4 bits or the network's type")
    args = parser.parse_args()
    model, tokens, rays, _ = train(args.steps, args.views, args.size, mixer=args.mixer,
                                   max_norm=args.max_norm)
    with torch.no_grad():
        whole = model(tokens, rays)
    streamed = stream(model, tokens, rays, args.cache_bits)
    off = max(float((whole[k] - streamed[k]).abs().max()) for k in whole)
    print(f"{tokens.shape[0]} tokens streamed one at a time: {streamed['mean'].shape[0]} splats, "
          f"largest difference from the whole stream's {off:.3f}")


if __name__ == "__main__":
    main()
