"""Waits inside the layer kernels that run out: the launch ends, the host is told, and the next launch is right.

Every wait is bounded and returns; the limit is set to no polls at all, so that waits for sums that take some time run out."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def operands(dtype, m, k, n):
    g = torch.Generator(device=DEV).manual_seed(m + k + n)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    return rand(m, k), rand(n, k), rand(n), rand(m, n)


@pytest.fixture
def shim():
    import __ash

    torch.cuda.synchronize()
    assert __ash.layer_timeouts(DEV) == 0
    yield __ash
    __ash.set_layer_wait_limit(-1)
    torch.cuda.synchronize()
    __ash.layer_timeouts(DEV)      # other tests find a count of their own


def calls():
    """(name, call): tiles that leave by bulk copies and by stores, with and without residuals, sums that are split, several
    phases, e4m3 rows, and the gradients' products.  Sums are long, so that none is there at the first poll."""
    import ash

    made = {}
    for dtype in (torch.float32, torch.bfloat16):
        for m, k, n in ((4096, 4096, 512), (2000, 4100, 130), (300, 40000, 128)):
            x, w, b, r = operands(dtype, m, k, n)
            made[f"{dtype} {m} {n}"] = lambda x=x, w=w, b=b: ash.fused_linear(x, w, b, "gelu")
            made[f"{dtype} {m} {n} residual"] = lambda x=x, w=w, b=b, r=r: ash.fused_linear(x, w, b, "silu", r)
        x, w, b, r = operands(dtype, 4096, 1024, 4096)
        made[f"{dtype} gradients"] = lambda x=x, w=w, b=b, r=r: ash.mlp.backend.linear_backward(r, None, 0, x, w, True, True, True)
    x, w, _, r = operands(torch.float32, 2048, 8192, 512)
    qx, qw = ash.quantize_rows(x), ash.quantize_rows(w)
    made["e4m3"] = lambda: ash.fused_linear(qx, qw, residual=r.bfloat16())
    return made


def test_a_wait_that_runs_out_is_told(shim):
    import ash

    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b)) if isinstance(a, tuple) else torch.equal(a, b)
    for name, call in calls().items():
        want = call()
        torch.cuda.synchronize()
        shim.set_layer_wait_limit(0)
        if "gradients" in name:      # its later products may find out about the first
            try:
                call()
            except RuntimeError as e:
                assert "ran out" in str(e), name
        else:
            call()
        shim.set_layer_wait_limit(-1)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="ran out"):      # the next call, whichever it is, without waiting
            call()
        with pytest.raises(RuntimeError, match="ran out"):      # and who asks
            ash.mlp.check_waits(DEV)
        assert same(call(), want), name                          # told once; launches are as they were
        ash.mlp.check_waits()
        assert shim.layer_timeouts(DEV) == 0


def test_a_replayed_graph_is_asked(shim):
    """A replay makes no call that could raise; check_waits does."""
    import ash

    x, w, b, _ = operands(torch.bfloat16, 4096, 4096, 512)
    want = ash.fused_linear(x, w, b)
    torch.cuda.synchronize()
    shim.set_layer_wait_limit(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ash.fused_linear(x, w, b)
    shim.set_layer_wait_limit(-1)
    graph.replay()
    with pytest.raises(RuntimeError, match="ran out"):
        ash.mlp.check_waits(0)
    assert torch.equal(ash.fused_linear(x, w, b), want)      # what was asked is not told again
    ash.mlp.check_waits("cuda")


def test_a_first_call_that_is_captured():
    """In a process of its own: the host's words are made inside the capture."""
    import subprocess
    import sys

    program = ("import torch, ash\n"
               "x, w = torch.ones(200, 64, device='cuda'), torch.ones(32, 64, device='cuda')\n"
               "torch.cuda.synchronize()\n"
               "g = torch.cuda.CUDAGraph()\n"
               "with torch.cuda.graph(g):\n"
               "    y = ash.fused_linear(x, w)\n"
               "g.replay()\n"
               "ash.mlp.check_waits()\n"
               "assert bool((y == 64).all())\n")
    import ash
    import os

    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(ash.__file__)))
    subprocess.run([sys.executable, "-c", program], env=env, check=True, timeout=300)
