"""The example that trains a readout on SOAP rows: every operator together."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

import train_readout  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda(cuda_device):
    yield


@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_fits_its_target(state_bits):
    losses, model, rows = train_readout.train(structures=32, steps=120, state_bits=state_bits)
    assert 0.8 < losses[0] < 1.2  # a standardised target, an untrained readout answers 0
    assert losses[-1] < 0.25 * losses[0]
    assert torch.isfinite(model.forward(rows)).all()


def test_training_repeats_bit_by_bit():
    first = train_readout.train(structures=8, steps=12)
    again = train_readout.train(structures=8, steps=12)
    for a, b in zip(first[1].parameters(), again[1].parameters()):
        assert torch.equal(a, b)


def test_readout_gradients_against_differences():
    """Gradients of the 8-bit readout against differences of the same network without rounding.

    Codes are off by at most 1/16 of themselves, independently of each other, and a gradient passes through four
    of them; over the thousands of terms of each sum such errors average out, so a tenth of the gradient's size is
    far above what rounding leaves and far below what a wrong formula gives."""
    batch = train_readout.workloads.config1(structures=4)
    rows = train_readout.soap_rows(batch)
    model = train_readout.Readout(rows.shape[1], blocks=1, seed=5)
    model.last["e"].normal_(generator=torch.Generator(device="cuda").manual_seed(7))
    weight = torch.randn(rows.shape[0], generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")

    def plain(parameters):
        g0, w, g1, up, down, g2, e = parameters

        def norm(x, g):
            return x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6) * g

        x = norm(rows.double(), g0) @ w.t()
        y = torch.nn.functional.silu(norm(x, g1) @ up.t()) @ down.t()
        return ((norm(x + y, g2) @ e) * weight).sum()

    model.forward(rows)
    grads = model.backward(weight)
    parameters = [p.double() for p in model.parameters()]
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").double()
        direction = direction + grad.double() * (direction.norm() / grad.double().norm())  # so that the slope is not small
        direction = direction / direction.norm()
        h = 1e-4
        ends = [plain([p + s * h * direction if j == i else p for j, p in enumerate(parameters)]) for s in (1.0, -1.0)]
        slope = float(ends[0] - ends[1]) / (2 * h)
        got = float((grad.double() * direction).sum())
        assert abs(got - slope) <= 0.1 * abs(slope), (i, got, slope)
