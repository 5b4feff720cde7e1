"""Memory that the Newton-Schulz iteration takes beside its inputs and results."""

import pytest
import torch

from packbalance_b200.ops.muon import muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
dev = "cuda"
GB = 1 << 30
BOUND = 2.1 * GB  # 2 GB of iterates, and the partial sums


def _peak(call):
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


def test_workspace_is_bounded():
    """A stack whose iterates would take several GB at once goes through in parts."""
    x = torch.randn(96, 2048, 2048, device=dev)
    got = []
    extra = _peak(lambda: got.append(orthogonalize(x))) - x.numel() * 2
    assert extra <= BOUND, f"{extra / GB:.2f} GB"
    for k in (0, 31, 95):  # the parts join without a seam
        assert torch.equal(orthogonalize(x[k : k + 1])[0], got[0][k])


def test_update_workspace_is_bounded():
    p = [torch.zeros(32, 2048, 2048, device=dev), torch.zeros(32, 1024, 4096, device=dev),
         torch.zeros(32, 4096, 1024, device=dev)]
    g, m = [torch.randn_like(t) for t in p], [torch.zeros_like(t) for t in p]
    extra = _peak(lambda: muon_update_(p, g, m, lr=0.01, weight_decay=0.0))
    assert extra <= BOUND, f"{extra / GB:.2f} GB"
    for t, h in zip(p, g):
        for k in (0, 17, 31):
            q, mom = torch.zeros_like(t[k]), torch.zeros_like(t[k])
            muon_update_([q], [h[k]], [mom], lr=0.01, weight_decay=0.0)
            assert torch.equal(q, t[k])


def test_one_matrix_beyond_the_bound():
    x = torch.randn(49152, 8192, device=dev).bfloat16()
    y = orthogonalize(x)
    assert y.shape == x.shape and bool(torch.isfinite(y).all())
    s = torch.linalg.matrix_norm(y.float()) / 8192**0.5  # singular values end between 0.7 and 1.2
    assert 0.7 < float(s) < 1.2
