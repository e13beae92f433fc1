"""A small matcher of padded keypoint sets, trained end to end on the GPU.

    descriptors -> linear -> group norm + silu -> linear -> group norm
                -> rotary positions (row, column) -> scores
                -> bidirectional softmax -> likelihood of the true matches

Every sample holds another number of keypoints; ``lengths`` keeps the padding
out of the norms' statistics and out of the softmaxes.  The second image of a
pair is the first one shifted, reordered and disturbed: descriptors alone leave
its repeated keypoints ambiguous, positions tell them apart.

    python examples/dense_matching.py [steps]
"""

from __future__ import annotations

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch
import torch.nn as nn

import dot


class Encoder(nn.Module):
    def __init__(self, inputs: int, channels: int = 64, groups: int = 8):
        super().__init__()
        self.inp = nn.Linear(inputs, channels)
        self.norm1 = dot.GroupNormAct(groups, channels, activation="silu")
        self.out = nn.Linear(channels, channels)
        self.norm2 = dot.GroupNormAct(groups, channels, activation="none")
        self.turn = dot.Rotary((channels // 4, channels // 4), theta=100.0)   # half the pairs for each axis

    def forward(self, x: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        x = self.norm1(self.inp(x), lengths)
        x = self.norm2(self.out(x), lengths)
        return self.turn(x.unsqueeze(-2), positions).squeeze(-2)


def matching(f0: torch.Tensor, f1: torch.Tensor, lengths: torch.Tensor, tau: float = 0.5) -> torch.Tensor:
    """Soft matching of two feature sets [N, L, C]: rows and columns normalised together."""
    scores = f0 @ f1.transpose(1, 2) / f0.size(-1) ** 0.5
    return dot.bidirectional_softmax(scores, tau=tau, lengths=torch.stack((lengths, lengths), dim=1))


def pairs(n: int, points: int, inputs: int, generator: torch.Generator, device="cuda"):
    """Two views of n keypoint sets: (descriptors, positions) each, the partner of every keypoint, lengths."""
    def rand(*shape):
        return torch.rand(*shape, generator=generator, device=device)

    lengths = (points // 2 + rand(n) * (points - points // 2)).to(torch.int32)
    kinds = torch.randn(6, inputs, generator=generator, device=device)           # few kinds: many look alike
    desc = kinds[(rand(n, points) * 6).long()]
    pos = rand(n, points, 2) * 30
    valid = torch.arange(points, device=device) < lengths[:, None]
    order = torch.argsort(torch.where(valid, rand(n, points), 2.0), dim=1)       # padding stays last
    noise = torch.randn(n, points, inputs, generator=generator, device=device)
    desc1 = torch.gather(desc, 1, order[..., None].expand_as(desc)) + noise
    pos1 = torch.gather(pos, 1, order[..., None].expand_as(pos)) + 4 * rand(n, 1, 2)
    return (desc, pos), (desc1, pos1), torch.argsort(order, dim=1), lengths


def train(steps: int = 200, seed: int = 0, report=None) -> list[float]:
    """Trains an encoder; returns the loss of every step."""
    torch.manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    model = Encoder(32).cuda()
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for step in range(steps):
        (d0, p0), (d1, p1), partner, lengths = pairs(8, 96, 32, gen)
        P = matching(model(d0, p0, lengths), model(d1, p1, lengths), lengths)
        valid = torch.arange(d0.size(1), device=d0.device) < lengths[:, None]
        hit = torch.gather(P, 2, partner[..., None]).squeeze(-1)[valid]
        loss = -torch.log(hit.clamp(min=1e-6)).mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and step % report == 0:
            right = (P.argmax(dim=2) == partner)[valid].float().mean()
            print(f"step {step:4d}  loss {float(loss.detach()):.3f}  matched {float(right):.2f}")
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 200, report=20)
