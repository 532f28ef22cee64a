"""Query/key norms: positions outside the tables under a partial rotation, outputs that share memory. Tolerances as
in test_qk_norm_gpu."""
from __future__ import annotations

import pytest
import torch
from test_qk_norm_gpu import DTYPES, U, close, make, reference, tables

from stagehand_amd.qk_norm import qk_norm_rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot", [(32, 16), (64, 64), (80, 32), (72, 36), (130, 34), (128, 2)])
def test_positions_outside_the_tables_give_nan_for_all_of_a_token(dim, rot, dtype, interleaved):
    """Also for the values that are not rotated, and in the gradients."""
    q, k, wq, wk = (t.requires_grad_() for t in make(2, 3, 1, 6, dim, dtype, seed=4))
    cos, sin = tables(10, rot)
    p = torch.tensor([[0, 9, 10, 3, -1, 2], [1, 2, 3, 2 ** 40, 5, -2 ** 40]], device="cuda")
    wrong = (p < 0) | (p >= 10)
    fine = torch.where(wrong, torch.zeros_like(p), p)
    outs = qk_norm_rope(q, k, wq, wk, cos, sin, positions=p, interleaved=interleaved)
    gs = [torch.randn_like(o) for o in outs]
    grads = torch.autograd.grad(outs, (q, k), gs)
    for y, x, w, g, dx in zip(outs, (q, k), (wq, wk), gs, grads):
        rows = wrong[:, None, :].expand(y.shape[:3])
        assert y[rows].isnan().all() and dx[rows].isnan().all()
        want, size, want_dx, size_dx, _, _ = reference(x, w, cos, sin, positions=fine, interleaved=interleaved, dy=g)
        keep = ~rows.cpu()
        close(y.detach().cpu()[keep], want[keep], 24 * U * size[keep], "y")
        close(dx.cpu()[keep], want_dx[keep], 48 * U * size_dx[keep], "dx")


def test_outputs_that_share_memory_are_refused():
    """Heads that several results would be written to."""
    q, k, wq, wk = make(2, 4, 2, 6, 64, torch.bfloat16)
    ko = torch.empty(k.shape, device="cuda", dtype=k.dtype)
    e = torch.empty(2 * 4 * 6 * 64, device="cuda", dtype=q.dtype)
    bad = [e[:64].expand(2, 4, 6, 64), e[:4 * 6 * 64].view(1, 4, 6, 64).expand(2, 4, 6, 64), e[:2 * 6 * 64].view(2, 1, 6, 64).expand(2, 4, 6, 64),
           e[:2 * 4 * 64].view(2, 4, 1, 64).expand(2, 4, 6, 64), e.as_strided((2, 4, 6, 64), (4 * 6 * 64, 6 * 64, 32, 1)),
           e.as_strided((2, 4, 6, 64), (64, 64, 64, 1))]
    for o in bad:
        with pytest.raises(ValueError, match="share memory"):
            qk_norm_rope(q, k, wq, wk, out=(o, ko))
    # one head or token: its stride does not matter
    one = torch.empty(1, 1, 6, 64, device="cuda", dtype=q.dtype).as_strided((1, 1, 6, 64), (0, 0, 64, 1))
    want, _ = qk_norm_rope(q[:1, :1], None, wq)
    assert torch.equal(qk_norm_rope(q[:1, :1], None, wq, out=(one, None))[0], want)
    # every order of the dims, gaps between heads
    want, _ = qk_norm_rope(q, None, wq)
    for order in ((0, 1, 2), (2, 1, 0), (1, 2, 0), (0, 2, 1)):
        shape = [q.shape[i] + (i == 1) for i in order]
        o = torch.empty(*shape, 70, device="cuda", dtype=q.dtype).permute(*[order.index(i) for i in range(3)], 3)[:, :4, :, 3:67]
        assert torch.equal(qk_norm_rope(q, None, wq, out=(o, None))[0], want)
    empty = torch.empty(0, device="cuda", dtype=q.dtype).as_strided((0, 4, 6, 64), (0, 0, 0, 1))
    qk_norm_rope(q[:0], None, wq, out=(empty, None))
