"""The gated block's operators together, as ``examples/gated_block.py`` runs them: training lowers the loss, and the
on-line run gives the whole-sequence outputs (float32 outputs of two orders of summation through two blocks and norms:
1e-4 of the largest value)."""

import importlib.util
from pathlib import Path

import pytest
import torch

_PATH = Path(__file__).resolve().parents[1] / "examples" / "gated_block.py"


def _example():
    spec = importlib.util.spec_from_file_location("gated_block_example", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _run(device):
    ex = _example()
    torch.manual_seed(0)
    model = ex.GatedModel(1, 1, width=48, heads=4, key_heads=2, key=8, value=12).to(device)
    losses = ex.train(model, 25, device, batch=8, length=130)
    assert sum(losses[-5:]) < 0.7 * sum(losses[:5])
    u, _ = ex.windows(3, 150, torch.Generator().manual_seed(1), device)
    with torch.no_grad():
        whole, states = model(u)
        first, carried = model(u[:, :70])
        second, carried = model(u[:, 70:], carried)
    bar = 1e-4 * float(whole.abs().max())
    assert (ex.online(model, u) - whole).abs().max() < bar
    assert (torch.cat((first, second), 1) - whole).abs().max() < bar
    for a, b in zip(states, carried):
        assert (a - b).abs().max() < 1e-4 * float(a.abs().max())
    return model, u


def test_example_on_the_cpu():
    _run("cpu")


@pytest.mark.gpu
def test_example_on_the_gpu(gpu):
    """And in bfloat16: the blocks' inputs rounded, the states float32."""
    model, u = _run(gpu)
    with torch.no_grad():
        want = model(u)[0]
        half = model.bfloat16()
        # decays and projections in bfloat16 throughout: some percent of the float32 model's outputs
        got, states = half(u.bfloat16())
    assert got.dtype == torch.bfloat16 and all(s.dtype == torch.float32 for s in states)
    assert (got.float() - want).abs().max() < 0.1 * want.abs().max()
