"""The example that runs the policy operators together (examples/policy_loop.py): it trains, and acting step by step over the caches
agrees with the window that training sees."""
import importlib.util
import math
from pathlib import Path

import pytest

from util import b2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
spec = importlib.util.spec_from_file_location("policy_loop", Path(__file__).resolve().parents[1] / "examples" / "policy_loop.py")


@pytest.fixture(scope="module")
def loop():
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_trains(loop):
    """Finite losses, gradients of every parameter, parameters that moved."""
    net, history, _ = loop.train(worlds=64, steps=20, iterations=3, say=lambda *a: None)
    assert len(history) == 3 and all(math.isfinite(v) for h in history for v in h.values())
    fresh = loop.Policy(net.enter.shape[1], 0)
    for p, q in zip(net.params, fresh.params):
        assert torch.isfinite(p).all() and not torch.equal(p, q)
    assert all(m.grad is not None and bool(m.grad.any()) for m in net.master)


def test_acting_agrees_with_the_window(loop):
    """Step by step over ragged caches and 8-bit weights against the whole window: the same network, so means that differ by the
    8-bit and 16-bit roundings only (each of the four 8-bit products is off by about 1% of its norm; both ways end within 5%)."""
    net, _, last = loop.train(worlds=48, steps=30, iterations=1, say=lambda *a: None)
    obs, first = last["obs"], last["first"]
    n, steps, _ = obs.shape
    caches = [tuple(torch.full((n, loop.EPISODE, loop.KV_HEADS, loop.DIM), math.nan, device="cuda", dtype=torch.bfloat16)
                    for _ in range(2)) for _ in range(loop.LAYERS)]
    with torch.no_grad():
        want = net.window(obs, first.contiguous())
    got = []
    for t in range(steps):
        got.append(net.act(obs[:, t], caches, (t - first[:, t] + 1).to(torch.int32)))
    got = torch.stack(got, 1)
    assert torch.isfinite(got).all()
    assert float((got - want).norm() / want.norm()) < 0.05
    assert (first > 0).any()  # episodes that began inside the window
