"""CPU: when the operators' scratch is kept (the CUDA runtime is replaced by what it would answer)."""
import pytest
import torch

from moe_swarm_b200 import ops


@pytest.fixture
def cuda(monkeypatch):
    """A process on device 0, stream 7, not capturing; scratch on the host."""
    state = dict(device=0, stream=7, capturing=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: state["stream"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: state["capturing"], raising=False)
    empty = torch.empty
    monkeypatch.setattr(ops.torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    monkeypatch.setattr(ops, "_scratch", {})
    return state


def test_small_scratch_is_kept_per_stream(cuda):
    first = ops._workspace(1000, 0)
    assert ops._workspace(2000, 0) is first
    cuda["stream"] = 8
    assert ops._workspace(2000, 0) is not first


@pytest.mark.parametrize("change", [dict(capturing=True), dict(device=1)])
def test_scratch_that_a_graph_may_hold_is_not_kept(cuda, change):
    """While a stream captures, and where that cannot be asked: on a device that is not the current one."""
    kept = ops._workspace(1000, 0)
    cuda.update(change)
    assert ops._workspace(1000, 0) is not kept
    assert len(ops._scratch) == 1


def test_large_scratch_is_not_kept(cuda):
    assert ops._workspace(ops._SCRATCH_KEPT + 1, 0).numel() == ops._SCRATCH_KEPT + 1 and not ops._scratch
