"""Captured training steps of the adapters' projection beside other graphs of the same leaves."""
import pytest
import torch

import moe_overlap_b200 as mo
from tests.test_lora_gpu import make

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")]


@pytest.fixture
def step(cuda_device):
    """Masters in fp32, and a step that casts them, projects and differentiates."""
    x, w, a, b, dy, scale, ids = make(200, 256, 320, 4, 16, torch.bfloat16, seed=1, device=cuda_device)
    masters = [a.float().requires_grad_(True), b.float().requires_grad_(True)]

    def run(wrt="masters"):
        low = [m.to(torch.bfloat16) for m in masters]
        y = mo.lora_linear(x, w, *low, ids, scale=scale)
        if wrt == "backward":
            for m in masters:
                m.grad = None
            y.backward(dy)
            return [m.grad for m in masters]
        return list(torch.autograd.grad(y, masters if wrt == "masters" else low, dy))

    run.masters = masters
    run.eager = lambda: mo.lora_linear(x, w, *(m.to(torch.bfloat16) for m in masters), ids, scale=scale)
    return run


def warm(step, wrt):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [g.clone() for g in step(wrt)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    return want


@pytest.mark.parametrize("wrt", ["masters", "backward", "low"])
def test_adapters_cast_from_masters_inside_the_capture(step, wrt):
    want = warm(step, wrt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(wrt)
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("wrt", ["masters", "backward"])
def test_a_graph_of_the_masters_from_before_is_refused(step, wrt):
    """... by the backward, which would come to their accumulators; the process and the GPU stay
    usable, and the same capture works once that graph is gone."""
    want = warm(step, wrt)
    alive = step.eager()
    with pytest.raises(RuntimeError, match="is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(wrt)
    torch.cuda.synchronize()
    assert bool(alive.isfinite().all())
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(wrt)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_a_pass_that_does_not_come_to_the_masters_is_captured_beside_it(step):
    want = warm(step, "low")
    alive = step.eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step("low")
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del alive


def test_a_held_accumulator_is_named_as_a_cause(cuda_device):
    """No graph of lora_linear is alive: something else holds a leaf's accumulator."""
    x, w, a, b, dy, scale, ids = make(40, 64, 72, 3, 8, torch.bfloat16, device=cuda_device)
    a.requires_grad_(True)
    held = a.expand_as(a).grad_fn.next_functions[0][0]
    with pytest.raises(RuntimeError, match="holds the accumulator"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(mo.lora_linear(x, w, a, b, ids, scale=scale), (a,), dy)
    torch.cuda.synchronize()
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (da,) = torch.autograd.grad(mo.lora_linear(x, w, a, b, ids, scale=scale), (a,), dy)
    graph.replay()
    (want,) = torch.autograd.grad(mo.lora_linear(x, w, a, b, ids, scale=scale), (a,), dy)
    assert torch.equal(da, want)
