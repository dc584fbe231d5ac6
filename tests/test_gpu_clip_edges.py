"""clip_grad_norm where two tensors share memory, and grad_norm, which may read some memory twice"""
import pytest
import torch

import spanqr_amd as sp

pytestmark = pytest.mark.gpu


def test_a_tensor_listed_twice(cuda):
    """in place, two workgroups would scale the same elements at once; read alone, or into two places, it counts twice"""
    a, b = torch.ones(3, 5, device=cuda), torch.ones(7, device=cuda)
    kept = a.clone()
    for twice in ([a, b, a], [a, a.view(-1)], [a, a[:1]]):
        with pytest.raises(ValueError, match="same memory"):
            sp.clip_grad_norm(twice, 1.0)
    with pytest.raises(ValueError, match="same memory"):
        sp.clip_grad_norm([a, kept], 1.0, out=[torch.empty_like(a)] * 2)
    assert torch.equal(a, kept)
    assert abs(float(sp.grad_norm([a, a])) - 30.0 ** 0.5) < 1e-6
    out = [torch.empty_like(a), torch.empty_like(a)]
    assert abs(float(sp.clip_grad_norm([a, a], 100.0, out=out)) - 30.0 ** 0.5) < 1e-6
    assert torch.equal(out[0], a) and torch.equal(out[1], a)
    # tensors without elements share nothing
    e = torch.empty(0, device=cuda)
    assert abs(float(sp.clip_grad_norm([e, e, a, torch.empty(0, 4, device=cuda)], 100.0)) - 15.0 ** 0.5) < 1e-6
