"""Fits several images with one model: a hash grid over the pixel coordinates, a latent code per image, a layer of experts that
share the work, and a fused network in front of the colour.

    coordinates -> FusedEncoding ----+
                                     +-> FusedLayerNorm -> FusedExperts (router, two layers each) -> FusedNetwork -> colour
    image number -> FusedEmbedding --+

The images are made up on the spot (waves of a frequency and a direction of their own). Run on a GPU:

    python examples/images_by_experts.py [--images 8] [--points 65536] [--steps 300]
"""
import argparse
import json
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "quick-mlp_b200"))

import torch  # noqa: E402

import qmlp  # noqa: E402
from qmlp import configs  # noqa: E402


class ImagesByExperts(torch.nn.Module):
    def __init__(self, images, code=16, hidden=64, width=32, experts=8, k=2):
        super().__init__()
        self.encoding = qmlp.FusedEncoding(json.dumps(configs.hashgrid(2, 8, 2, 12, 4, 256)))
        self.grid = torch.nn.Parameter(self.encoding.create_parameter_tensor().cuda() * 0.1)
        self.codes = qmlp.FusedEmbedding(images, code, scale=code ** 0.5)
        channels = self.encoding.num_output_channels() + code
        self.norm = qmlp.FusedLayerNorm(channels)
        self.experts = qmlp.FusedExperts(channels, hidden, width, experts, k)
        self.head = qmlp.FusedNetwork(json.dumps(configs.identity_net(width, [32, 1], ["relu", "identity"])), weight_dtype=torch.float32)

    def forward(self, points, image):
        features = torch.cat([self.encoding(points, self.grid), self.codes(image)], dim=1)
        return self.head(self.experts(self.norm(features)).float())


def colour(points, image):
    """one wave per image"""
    angle = image.float() * 0.7
    along = points[:, 0] * torch.cos(angle) + points[:, 1] * torch.sin(angle)
    return 0.5 + 0.5 * torch.sin((4 + image.float()) * along)[:, None]


def fit(images=8, points=65536, steps=300, seed=0, report=print):
    """mean squared errors of the steps"""
    torch.manual_seed(seed)
    model = ImagesByExperts(images)
    optimizer = torch.optim.Adam(model.parameters(), lr=5e-3)
    losses = []
    for step in range(steps):
        x = torch.rand((points, 2), device="cuda")
        image = torch.randint(images, (points,), device="cuda")
        loss = torch.nn.functional.mse_loss(model(x, image), colour(x, image))
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report is not None and (step % 50 == 0 or step == steps - 1):
            report(f"step {step}: mean squared error {loss.item():.5f}")
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--images", type=int, default=8)
    parser.add_argument("--points", type=int, default=65536)
    parser.add_argument("--steps", type=int, default=300)
    a = parser.parse_args()
    fit(a.images, a.points, a.steps)
