"""AttentionBlock with decays of its own."""
import pytest
import torch

import blockcheck as bc
from lfcheck import TORCH_DT, gen
from test_gpu_gated_norm import _plain_block

pytestmark = pytest.mark.gpu

OWN = [-0.25, -0.004, -2.0]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_own_decays_through_a_state_dict(gpu, dtype):
    """A block with decays of its own, saved, loaded into one that was built with the defaults, and run: against the plain form, in
    test_blocks_together's norm-relative bounds for one block, 44 u (fp32: 400 u)."""
    import laplacianformer_amd as lf

    print(f"decay block {dtype}", flush=True)
    torch.manual_seed(21)
    t = TORCH_DT[dtype]
    B, N, C = 2, 75, 96
    own = lf.AttentionBlock(C, 3, attention="decay", log_decay=OWN).to(t)
    lengths = torch.tensor([N, N - 20], dtype=torch.int32)
    x = gen((B, N, C), 80, dtype)
    want, total, _ = _plain_block(own, x.double(), None, None, lengths, True)
    block = lf.AttentionBlock(C, 3, attention="decay").to(t).to(gpu)
    block.load_state_dict(own.state_dict())
    assert block._log_decay.device.type == "cuda" and torch.equal(block._log_decay.cpu(), torch.tensor(OWN))
    with torch.no_grad():
        y, s = block(x.to(gpu), lengths=lengths.to(gpu))
    u = bc.unit(t) * (400 if dtype == "f32" else 44)
    assert (y.cpu().double() - want).norm() <= u * want.norm() and torch.equal(s.cpu(), x)
    with torch.no_grad():
        other = lf.AttentionBlock(C, 3, attention="decay").to(t)
        other.load_state_dict({n: p for n, p in own.state_dict().items() if n != "_log_decay"} | {"_log_decay": other._log_decay})
        z, _ = other.to(gpu)(x.to(gpu), lengths=lengths.to(gpu))
    assert (z.cpu().double() - want).norm() > 2 * u * want.norm()  # so that the first assertion tells the two apart


def test_first_call_captured(gpu):
    """A block's first call may be one under capture: nothing is moved to the GPU in it."""
    import laplacianformer_amd as lf

    torch.manual_seed(22)
    a, b = (lf.AttentionBlock(64, 2, attention="decay", positions=False).to(gpu) for _ in range(2))
    b.load_state_dict(a.state_dict())
    x = gen((1, 40, 64), 81, "f32").to(gpu)
    with torch.no_grad():
        want = a(x)[0]  # the libraries' handles exist from here on; block b has not run
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b(x)[0]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            a(x)
