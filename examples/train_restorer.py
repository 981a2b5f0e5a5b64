"""One training step after another of a small window-attention restoration network:
the framework's loss, its attention with a learned relative position bias, and its
orthogonalised weight updates, together.

    python examples/train_restorer.py [--steps 20] [--size 64] [--batch 4] [--device cuda]

The network removes noise from synthetic images: patches become tokens, two blocks
attend in (shifted) 8 x 8 windows with ``fa.relative_attention``, and ``1 - fa.ssim``
is the loss.  Matrices are updated with momentum through ``fa.orthogonalize``, the
rest (biases, norms, bias tables) by plain gradient steps.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import frame_analytics_amd as fa  # noqa: E402

WINDOW = 8


def cut(x, shift):
    """(n, h, w, c) -> (n * windows, 64, c), the frame rolled by ``shift`` first."""
    n, h, w, c = x.shape
    x = torch.roll(x, (-shift, -shift), dims=(1, 2)) if shift else x
    x = x.view(n, h // WINDOW, WINDOW, w // WINDOW, WINDOW, c).transpose(2, 3)
    return x.reshape(-1, WINDOW * WINDOW, c)


def join(x, n, h, w, shift):
    x = x.view(n, h // WINDOW, w // WINDOW, WINDOW, WINDOW, -1).transpose(2, 3)
    x = x.reshape(n, h, w, -1)
    return torch.roll(x, (shift, shift), dims=(1, 2)) if shift else x


def shift_mask(h, w, shift, device):
    """(windows, 1, 64, 64): tokens of a rolled frame that were neighbours."""
    def part(size):
        at = torch.arange(size, device=device)
        return (at >= size - WINDOW).int() + (at >= size - shift).int()

    region = 3 * part(h)[:, None] + part(w)[None, :]
    r = cut(region[None, :, :, None], 0)[..., 0]
    return (r[:, None, :, None] == r[:, None, None, :]).contiguous()


class Block(nn.Module):
    def __init__(self, dim, heads, shift):
        super().__init__()
        self.heads, self.shift = heads, shift
        self.positions = fa.GridPositions(WINDOW, WINDOW)
        self.norm1, self.norm2 = nn.LayerNorm(dim), nn.LayerNorm(dim)
        self.qkv, self.out = nn.Linear(dim, 3 * dim), nn.Linear(dim, dim)
        self.up, self.down = nn.Linear(dim, 2 * dim), nn.Linear(2 * dim, dim)
        self.table = nn.Parameter(torch.zeros(self.positions.rows, heads))

    def forward(self, x):
        n, h, w, c = x.shape
        tokens = cut(self.norm1(x), self.shift)
        # (windows, 64, 3, heads, dim) -> three views of (windows, heads, 64, dim)
        q, k, v = self.qkv(tokens).view(*tokens.shape[:2], 3, self.heads, -1).permute(2, 0, 3, 1, 4)
        mask = shift_mask(h, w, self.shift, x.device) if self.shift else None
        a = fa.relative_attention(q, k, v, self.table, self.positions, mask=mask)
        x = x + join(self.out(a.transpose(1, 2).reshape(tokens.shape)), n, h, w, self.shift)
        return x + self.down(F.gelu(self.up(self.norm2(x))))


class Restorer(nn.Module):
    def __init__(self, dim=60, heads=2):
        super().__init__()
        self.first = nn.Conv2d(3, dim, 3, padding=1)
        self.blocks = nn.ModuleList([Block(dim, heads, 0), Block(dim, heads, WINDOW // 2)])
        self.last = nn.Conv2d(dim, 3, 3, padding=1)

    def forward(self, x):
        y = self.first(x).permute(0, 2, 3, 1)
        for block in self.blocks:
            y = block(y)
        return x + self.last(y.permute(0, 3, 1, 2))


@torch.no_grad()
def update(net, momentum, lr=0.001, beta=0.9):
    for name, p in net.named_parameters():
        m = momentum.setdefault(name, torch.zeros_like(p))
        m.mul_(beta).add_(p.grad)
        if p.ndim >= 2 and not name.endswith("table"):
            flat = m.reshape(p.shape[0], -1)
            step = fa.orthogonalize(flat).reshape(p.shape)
            p.sub_(step, alpha=lr * 0.2 * max(flat.shape) ** 0.5)
        else:
            p.sub_(m, alpha=lr)
        p.grad = None


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--size", type=int, default=64)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    net, momentum, losses = Restorer().to(a.device), {}, []
    for i in range(a.steps):
        clean = F.interpolate(torch.rand(a.batch, 3, 9, 9, device=a.device), size=a.size,
                              mode="bicubic", align_corners=False).clamp(0, 1)
        noisy = clean + 0.1 * torch.randn_like(clean)
        loss = 1.0 - fa.ssim(net(noisy), clean, data_range=1.0)
        loss.backward()
        update(net, momentum)
        losses.append(loss.item())
        print(f"step {i}: 1 - ssim = {losses[-1]:.4f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
