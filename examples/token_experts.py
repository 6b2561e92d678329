"""A field per object, learned with the operators on tokens in front of a coordinate network.

Every object has a token. Its learned code (embedding) is normalised (layer norm) and refined by experts: a router picks two of
them per token (route), the tokens are sorted by expert (group), go to their places there (dispatch), through the experts' linear
layers, with one of the framework's activations in between, and back (combine). A fused coordinate network decodes the code and a
position to the value of the field there. Once trained, the experts are served with weights of 4 bits.

    python examples/token_experts.py [steps]
"""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quick-mlp_amd"))
import qmlp  # noqa: E402
from qmlp import tokens  # noqa: E402


class Experts(torch.nn.Module):
    """Each token's two experts of a layer, weighted by the router's probabilities, on top of the token itself."""

    def __init__(self, experts, channels, hidden, chosen=2):
        super().__init__()
        self.count, self.chosen = experts, chosen
        self.norm = qmlp.FusedLayerNorm(channels)
        self.router = torch.nn.Linear(channels, experts, bias=False, device="cuda")
        self.first = qmlp.FusedGroupedLinear(experts, channels, hidden)
        self.activation = qmlp.FusedActivation("celu")
        self.second = qmlp.FusedGroupedLinear(experts, hidden, channels)

    def forward(self, x):
        normal = self.norm(x)
        weights, experts = tokens.route(self.router(normal), self.chosen)
        # the rows (token, choice) by expert, and where each of them goes
        _, offsets, places = tokens.group(experts, self.count, places=True)
        rows = tokens.dispatch(normal.half(), places)   # in 16 bits, as the activation works
        rows = self.second(self.activation(self.first(rows, offsets)), offsets)
        return tokens.combine(rows.to(x.dtype), places, weights, x)

    def quantise(self):
        """For serving: the experts' weights in 4 bits."""
        self.first, self.second = (qmlp.FusedMx4GroupedLinear(layer) for layer in (self.first, self.second))


class ObjectFields(torch.nn.Module):
    def __init__(self, objects, channels=32, experts=8, hidden=64):
        super().__init__()
        self.codes = qmlp.FusedEmbedding(objects, channels, scale=channels ** 0.5)
        with torch.no_grad():
            self.codes.table.mul_(channels ** -0.5)
        self.experts = Experts(experts, channels, hidden)
        identity = {"id": "identity", "start_in": 0, "n_in": 3 + channels}
        layer = {"n_out": 64, "bias": True, "activation": "relu"}
        self.decoder = qmlp.FusedNetwork(json.dumps({
            "num_inputs": 3 + channels, "num_outputs": 1, "activation_specification": ["qmlp/builtin-activations.json"],
            "encodings": [identity], "network": [layer, layer, {"n_out": 1, "bias": True, "activation": "identity"}]}),
            weight_dtype=torch.float32)

    def forward(self, objects, positions):
        """The fields of the objects (B) at their positions (B, P, 3): (B, P)."""
        codes = self.experts(self.codes(objects))
        inputs = torch.cat([2 * positions - 1, codes[:, None, :].expand(-1, positions.shape[1], -1)], 2)
        return self.decoder(inputs.reshape(-1, inputs.shape[2])).view(positions.shape[:2])


def balls(objects):
    """Centres and radii."""
    return torch.rand(objects, 3, device="cuda"), 0.1 + 0.3 * torch.rand(objects, device="cuda")


def batch_of(centres, radii, batch, points):
    """Objects, positions and the signed distances there."""
    index = torch.randint(0, len(radii), (batch,), device="cuda")
    positions = torch.rand(batch, points, 3, device="cuda")
    return index, positions, (positions - centres[index][:, None]).norm(dim=2) - radii[index][:, None]


def fit(model, centres, radii, steps, batch=256, points=64):
    """Returns the losses."""
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-2)
    losses = []
    for _ in range(steps):
        index, positions, target = batch_of(centres, radii, batch, points)
        loss = (model(index, positions) - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def train(steps=300, objects=500, batch=256, points=64, seed=0):
    """Fits balls of different places and sizes (signed distances); returns the losses."""
    torch.manual_seed(seed)
    shapes = balls(objects)
    return fit(ObjectFields(objects), *shapes, steps, batch, points)


if __name__ == "__main__":
    torch.manual_seed(0)
    shapes = balls(500)
    model = ObjectFields(500)
    history = fit(model, *shapes, int(sys.argv[1]) if len(sys.argv) > 1 else 300)
    for step in range(0, len(history), max(1, len(history) // 10)):
        print("step %4d: mean squared error %.5f" % (step, history[step]))
    print("step %4d: mean squared error %.5f" % (len(history) - 1, history[-1]))
    with torch.no_grad():
        index, positions, target = batch_of(*shapes, 500, 256)
        for name in ("as they are", "in 4 bits"):
            if name == "in 4 bits":
                model.experts.quantise()
            print("experts' weights %s: %.5f" % (name, (model(index, positions) - target).square().mean()))
