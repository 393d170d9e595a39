"""install_linears on the GPU: what it holds, on which streams and in which graphs it runs."""
import copy

import pytest
import torch

from tests.test_router_layer_gpu import rel_err

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_weights_that_leave_the_gpu_are_not_held(lib):
    from promoe_b200.hf_fused import install_linears
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    m = torch.nn.Sequential(*(torch.nn.Linear(1024, 1024) for _ in range(4))).to(BF16).cuda().requires_grad_(False)
    assert install_linears(m) == 4
    x = torch.randn(3, 1024).to(BF16)
    y = m(x.cuda()).cpu()
    assert torch.cuda.memory_allocated() - before >= 4 * 2 * 1024 * 1024
    m.cpu()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < 1024 * 1024
    assert rel_err(m(x), y) < 3e-2  # four roundings to bf16 on each side
    m.cuda()
    assert torch.equal(m(x.cuda()).cpu(), y)


def test_another_stream_and_a_graph(lib):
    from promoe_b200.hf_fused import install_linears
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.SiLU(), torch.nn.Linear(96, 64)).to(BF16).cuda().requires_grad_(False)
    own = copy.deepcopy(m).double()
    install_linears(m)
    x = torch.randn(5, 64, device="cuda").to(BF16)
    want = own(x.double())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = m(x)
    torch.cuda.current_stream().wait_stream(s)
    assert rel_err(y, want) < 1e-2
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(x)
    x.mul_(-1.0)
    g.replay()
    torch.cuda.synchronize()
    assert rel_err(y, own(x.double())) < 1e-2
