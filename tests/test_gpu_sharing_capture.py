"""GPU tests of sharing enabled after a graph was captured that does not know of it: refused,
since its replays would give blocks to the ring that others hold, or write to them."""

import pytest
import torch

import vpa
from tests._util import u32

pytestmark = pytest.mark.gpu


def allocator(device):
    a = vpa.DeviceBlockAllocator(20, 8, 4, 4, device)
    target = u32([20, 9, 0, 0], device)
    a.allocate(target)
    a.positions.copy_(target)
    return a, [torch.zeros((20, 4), device=device)]


def calls(a, device):
    keep = u32([99, 99, 99, 99], device)
    tokens = u32([20, 9, 0, 0], device)
    finished = torch.tensor([0, 0, 1, 1], dtype=torch.uint8, device=device)
    return {"release": lambda: a.release(keep), "trim": lambda: a.trim(tokens), "step": lambda: a.step(finished)}


@pytest.mark.parametrize("name", ["release", "trim", "step"])
def test_a_graph_captured_before(device, name):
    a, pool = allocator(device)
    call = calls(a, device)[name]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for enable in (a.enable_sharing, lambda: a.fork(u32([0], device), u32([2], device), pool)):
        with pytest.raises(vpa.VpaError, match="captured"):
            enable()
    assert a.shared is None
    # rows of their own go on
    graph.replay()
    a.step()
    torch.cuda.synchronize()
    assert int(a.positions[0]) >= 20


@pytest.mark.parametrize("name", ["release", "trim", "step"])
def test_eager_calls_before(device, name):
    a, pool = allocator(device)
    calls(a, device)[name]()
    assert a.fork(u32([0], device), u32([3], device), pool).cpu().all()
    assert int(a.shared.view(torch.int32).sum()) == 2


def test_another_allocator_s_graph(device):
    a, pool = allocator(device)
    b, _ = allocator(device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    assert a.fork(u32([0], device), u32([2], device), pool).cpu().all()
