"""Energies and forces of structures from an attention model over their nodes.

    python examples/structure_energy.py [--structures 64] [--pretrain 0] [--steps 20] [--bf16]

Kinds are embedded, a few layers of attention (with distances) and gated feed-forward blocks mix the nodes of each structure,
one learnable query for each structure reads the energy out, and the forces are its gradient with respect to the positions.
``--pretrain`` first takes that many steps on hidden kinds: some nodes' kinds are not shown, and the model is asked for them.
Training fits energies and forces of a pair potential, so a step differentiates the attention twice; ``--bf16`` then evaluates
the energies once more with 16-bit operands."""
import argparse
import os
import sys
from typing import Optional

import torch
from torch import Tensor, nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from equitorch_amd.nn import AddRMSNorm, Embedding, GatedFeedForward, KindCrossEntropy, SegmentAttention  # noqa: E402
from equitorch_amd.nn.functional import AttentionPlan  # noqa: E402
from equitorch_amd.optim import AdamW  # noqa: E402


class Layer(nn.Module):
    """Norm, attention, norm, feed-forward.  ``(update, x)``: what the layer before adds to ``x`` and ``x``, the sum of the layers'
    results, which stays in fp32; a norm adds the one to the other."""

    def __init__(self, channels: int, heads: int, kv_heads: int, hidden: int):
        super().__init__()
        self.norm1, self.norm2 = AddRMSNorm(channels), AddRMSNorm(channels)
        self.attention = SegmentAttention(channels, heads, kv_heads, cap=30.0)
        self.feed_forward = GatedFeedForward(channels, hidden)

    def forward(self, update: Tensor, x: Optional[Tensor], plan: AttentionPlan, pos: Tensor):
        dtype = self.attention.weight_in.dtype
        out, x = self.norm1(update, x)
        out, x = self.norm2(self.attention(out.to(dtype), plan, pos), x)
        return self.feed_forward(out.to(dtype)), x


class StructureEnergy(nn.Module):
    """``(kind (N,), pos (N, 3), ptr (S + 1,)) -> energies (S,)``."""

    def __init__(self, kinds: int = 8, channels: int = 64, heads: int = 4, kv_heads: int = 2, hidden: int = 128, layers: int = 2):
        super().__init__()
        self.embedding = Embedding(kinds, channels)
        self.layers = nn.ModuleList(Layer(channels, heads, kv_heads, hidden) for _ in range(layers))
        self.norm = AddRMSNorm(channels)
        self.query = nn.Parameter(torch.randn(1, channels))
        self.readout = SegmentAttention(channels, heads, kv_heads, distances=False)
        self.head = nn.Linear(channels, 1)

    def operands(self, dtype: torch.dtype) -> "StructureEnergy":
        """Rounds the weights of attention and feed-forward blocks; norms, sums and the head stay in fp32."""
        for module in self.modules():
            if isinstance(module, (SegmentAttention, GatedFeedForward)):
                module.to(dtype)
        return self

    def nodes(self, kind: Tensor, pos: Tensor, ptr: Tensor) -> Tensor:
        """Features of every node, the sum of the layers' results after a norm; a kind of -1 is embedded as zeros."""
        plan = AttentionPlan(ptr)
        update, x = self.embedding(kind), None
        for layer in self.layers:
            update, x = layer(update, x, plan, pos)
        return self.norm(update, x)[0]

    def forward(self, kind: Tensor, pos: Tensor, ptr: Tensor) -> Tensor:
        each = AttentionPlan(torch.arange(len(ptr), device=ptr.device), ptr)       # one query for each structure
        dtype = self.readout.weight_in.dtype
        query = self.query.expand(len(ptr) - 1, -1).to(dtype)
        out = self.readout(query, each, x_k=self.nodes(kind, pos, ptr).to(dtype))
        return self.head(out.float())[:, 0] * torch.diff(ptr)

    def energy_and_forces(self, kind: Tensor, pos: Tensor, ptr: Tensor, create_graph: bool = False):
        pos = pos.detach().requires_grad_(True)
        energy = self(kind, pos, ptr)
        (grad,) = torch.autograd.grad(energy.sum(), pos, create_graph=create_graph)
        return energy, -grad


def pair_potential(kind: Tensor, pos: Tensor, ptr: Tensor):
    """Energies and forces of soft pairs whose strength goes by the kinds: what the model is fitted to."""
    pos = pos.detach().requires_grad_(True)
    strength = 1.0 + 0.25 * kind.float()
    energies = []
    for a, b in zip(ptr[:-1].tolist(), ptr[1:].tolist()):
        d2 = (pos[a:b, None] - pos[None, a:b]).square().sum(-1)
        energies.append((strength[a:b, None] * strength[None, a:b] * torch.exp(-d2)).triu(1).sum())
    energy = torch.stack(energies)
    (grad,) = torch.autograd.grad(energy.sum(), pos)
    return energy.detach(), -grad


def make_structures(structures: int, generator: torch.Generator, device):
    """Random structures of 5 to 40 nodes: ``(kind, pos, ptr)``."""
    sizes = torch.randint(5, 41, (structures,), generator=generator)
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    kind = torch.randint(0, 8, (int(ptr[-1]),), generator=generator)
    pos = torch.randn(int(ptr[-1]), 3, generator=generator) * 2.0
    return kind.to(device), pos.to(device), ptr.to(device)


def hidden_kinds_loss(model: StructureEnergy, loss: KindCrossEntropy, data, hidden: Tensor) -> Tensor:
    """Mean cross entropy of the kinds of the ``hidden`` nodes, which the model does not see."""
    kind, pos, ptr = data
    shown, asked = kind.masked_fill(hidden, -1), kind.masked_fill(~hidden, -1)
    return loss(model.nodes(shown, pos, ptr).to(loss.weight.dtype), asked).sum() / hidden.sum().clamp(min=1)


def pretrain(model: StructureEnergy, data, steps: int, share: float = 0.15, report=None):
    """Asks for the kinds of a share of the nodes, another in every step, scored against the embedding's own table; states of the
    optimizer in 8 bits.  Returns the loss of every step."""
    table = model.embedding.weight
    loss = KindCrossEntropy(*table.shape).to(table.device)
    loss.weight = table
    optimizer = AdamW([p for n, p in model.named_parameters() if not n.startswith(("query", "readout", "head"))], lr=2e-3, state_bits=8)
    losses = []
    for step in range(steps):
        value = hidden_kinds_loss(model, loss, data, torch.rand(len(data[0]), device=table.device) < share)
        optimizer.zero_grad()
        value.backward()
        optimizer.step()
        losses.append(value.detach())
        if report is not None:
            report(step, float(losses[-1]))
    return torch.stack(losses)


def train(model: StructureEnergy, data, steps: int, report=None):
    """Fits energies (a node) and forces; returns the loss of every step."""
    kind, pos, ptr = data
    energy, forces = pair_potential(*data)
    optimizer = AdamW(model.parameters(), lr=2e-3, weight_decay=0.0)
    losses = []
    for step in range(steps):
        e, f = model.energy_and_forces(kind, pos, ptr, create_graph=True)
        loss = ((e - energy) / torch.diff(ptr)).square().mean() + (f - forces).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report is not None:
            report(step, float(losses[-1]))
    return torch.stack(losses)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--structures", type=int, default=64)
    parser.add_argument("--pretrain", type=int, default=0)
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--bf16", action="store_true")
    args = parser.parse_args()
    device = torch.device("cuda")
    torch.manual_seed(0)
    data = make_structures(args.structures, torch.Generator().manual_seed(0), device)
    model = StructureEnergy().to(device)
    if args.pretrain:
        pretrain(model, data, args.pretrain, report=lambda step, loss: print(f"pretraining step {step}: loss {loss:.5f}", flush=True))
    train(model, data, args.steps, lambda step, loss: print(f"step {step}: loss {loss:.5f}", flush=True))
    with torch.no_grad():
        energy = model(*data)
        print("energies", energy[:4].tolist())
        if args.bf16:
            print("with bf16 operands", model.operands(torch.bfloat16)(*data)[:4].tolist())


if __name__ == "__main__":
    main()
