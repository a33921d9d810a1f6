"""Train a readout on SOAP rows, then answer for one structure.

The rows of a batch of periodic cells (configuration 1: 64 atoms, two species,
144 features) are computed on the GPU and never leave it.  A residual network
with 8-bit products maps each atom's row to an energy; the sum over a
structure's atoms is fitted to a target by AdamW with 8-bit states:

    python examples/train_readout.py [--structures 64] [--steps 200] [--state-bits 8]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from mdescriptor_b200 import readout, workloads  # noqa: E402
from mdescriptor_b200.soap import Soap, device_view  # noqa: E402


def soap_rows(batch, device: int = 0) -> torch.Tensor:
    """float32 rows [atoms, features] of a batch, on the device."""
    cfg = workloads.CONFIGS[1]
    soap = Soap(cfg.species, r_cut=cfg.r_cut, n_max=cfg.n_max, l_max=cfg.l_max, average="off", dtype="float32")
    held = [torch.from_numpy(a).to(f"cuda:{device}") for a in (batch.numbers, batch.positions, batch.cells, batch.pbc, batch.offsets)]
    rows = torch.empty(int(batch.offsets[-1]), soap.feature_count, device=f"cuda:{device}")
    stream = torch.cuda.current_stream(device).cuda_stream
    view = device_view(*[t.data_ptr() for t in held], len(batch.offsets) - 1, int(batch.offsets[-1]))
    soap.compute_device(view, rows.data_ptr(), device, stream)
    soap.check(device, stream)
    return rows


class Readout:
    """Per-atom energies from rows: norm and first product, then residual
    blocks of norm, product, SiLU, product, and a last norm with one weight a
    channel.  Weights are float32; each step lays them out in 8 bits, as they
    are (for the products) and transposed (for the gradients)."""

    def __init__(self, features: int, width: int = 128, hidden: int = 256, blocks: int = 2, seed: int = 0) -> None:
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def weight(n: int, k: int) -> torch.Tensor:
            return torch.randn(n, k, generator=g, device="cuda") * k ** -0.5

        def ones(n: int) -> torch.Tensor:
            return torch.ones(n, device="cuda")

        self.first = {"g": ones(features), "w": weight(width, features)}
        self.blocks = [{"g": ones(width), "up": weight(hidden, width), "down": weight(width, hidden) * 0.5} for _ in range(blocks)]
        self.last = {"g": ones(width), "e": torch.zeros(width, device="cuda")}
        self.layout()

    def parameters(self) -> list[torch.Tensor]:
        return [p for part in (self.first, *self.blocks, self.last) for p in part.values()]

    def layout(self) -> None:
        """The 8-bit forms of the weights; after every change of them."""
        self.w = readout.quantize(self.first["w"], layout="tiles")
        self.up = [readout.quantize(b["up"], layout="tiles") for b in self.blocks]
        self.down = [readout.quantize(b["down"], layout="tiles") for b in self.blocks]

    def forward(self, rows: torch.Tensor) -> torch.Tensor:
        """Energies [atoms]; what the gradient needs is kept until ``backward``."""
        n = readout.rms_norm(rows, self.first["g"], output="float8")
        self.kept = [n]
        stream, branch = None, readout.matmul(n.output, self.w.rows)
        for block, up, down in zip(self.blocks, self.up, self.down):
            n = readout.rms_norm(branch, block["g"], residual=stream, output="float8")
            h = readout.matmul(n.output, up.rows)
            a = torch.nn.functional.silu(h)
            stream, branch = n.sum, readout.matmul(readout.quantize(a).rows, down.rows)
            self.kept.append((n, h, a))
        n = readout.rms_norm(branch, self.last["g"], residual=stream)
        self.kept.append(n)
        return n.output.float() @ self.last["e"]

    def backward(self, d_energy: torch.Tensor) -> list[torch.Tensor]:
        """Gradients, in the order of ``parameters``, from that of the energies."""
        n = self.kept.pop()
        d_e = n.output.float().t() @ d_energy
        d_out = (d_energy[:, None] * self.last["e"]).to(torch.bfloat16)
        d, d_g = readout.rms_norm_backward(d_out, n.sum, n.rstd, self.last["g"])
        grads = [d_g, d_e]
        for block, up, down in zip(reversed(self.blocks), reversed(self.up), reversed(self.down)):
            n, h, a = self.kept.pop()
            d8, a8 = readout.quantize(d, layout="both"), readout.quantize(a, layout="columns")
            d_down = readout.matmul(d8.columns, a8.columns, dtype="float32")
            d_a = readout.matmul(d8.rows, down.columns).float()
            sig = torch.sigmoid(h.float())
            d_h = (d_a * sig * (1.0 + h.float() * (1.0 - sig))).to(torch.bfloat16)
            d8 = readout.quantize(d_h, layout="both")
            x8 = readout.quantize(n.sum, layout="columns", row_factor=n.rstd, col_factor=block["g"])
            d_up = readout.matmul(d8.columns, x8.columns, dtype="float32")
            d, d_g = readout.rms_norm_backward(readout.matmul(d8.rows, up.columns), n.sum, n.rstd, block["g"], dsum=d)
            grads = [d_g, d_up, d_down] + grads
        n = self.kept.pop()
        d8 = readout.quantize(d, layout="both")
        x8 = readout.quantize(n.sum, layout="columns", row_factor=n.rstd, col_factor=self.first["g"])
        d_w = readout.matmul(d8.columns, x8.columns, dtype="float32")
        d_rows = readout.matmul(d8.rows, self.w.columns, dtype="float32")
        _, d_g = readout.rms_norm_backward(d_rows, n.sum, n.rstd, self.first["g"])
        return [d_g, d_w] + grads


def train(structures: int = 64, steps: int = 200, state_bits: int = 8, seed: int = 0) -> tuple[list[float], Readout, torch.Tensor]:
    """(loss of each step, the readout, rows of the last structure)."""
    batch = workloads.config1(structures=structures)
    rows = soap_rows(batch)
    offsets = torch.from_numpy(batch.offsets).cuda()
    of_structure = torch.repeat_interleave(torch.arange(structures, device="cuda"), offsets[1:] - offsets[:-1])
    # the target: a smooth function of every atom's row, summed over its structure and standardised
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    unit = rows / rows.norm(dim=1, keepdim=True)
    atom = torch.tanh(3.0 * (unit - unit.mean(0)) @ torch.randn(rows.shape[1], generator=g, device="cuda"))
    target = torch.segment_reduce(atom, "sum", offsets=offsets)
    target = (target - target.mean()) / target.std()
    per_atom = structures / rows.shape[0]  # a structure's answer is the mean over its atoms
    model = Readout(rows.shape[1], seed=seed)
    optimizer = readout.AdamW(model.parameters(), lr=3e-3, state_bits=state_bits, seed=seed)
    losses = []
    for _ in range(steps):
        energy = torch.segment_reduce(model.forward(rows), "sum", offsets=offsets) * per_atom
        miss = energy - target
        losses.append((miss * miss).mean())
        optimizer.step(model.backward((2.0 / structures * per_atom) * miss[of_structure]))
        model.layout()
    readout.check()
    return [float(v) for v in losses], model, rows[int(offsets[-2]):]


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--structures", type=int, default=64)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = parser.parse_args()
    losses, model, rows = train(args.structures, args.steps, args.state_bits)
    for step in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {step:5d}  mean squared error {losses[step]:.4f}")
    print(f"step {len(losses) - 1:5d}  mean squared error {losses[-1]:.4f}")
    energy = model.forward(rows)
    print(f"one structure of {rows.shape[0]} atoms: {float(energy.mean()):.4f}")


if __name__ == "__main__":
    main()
