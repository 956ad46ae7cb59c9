"""ops.orthogonalise over its whole range: norms, eps and coefficients far from the usual ones, classes of sizes that the
other tests do not reach, and refusals."""
import pytest
import torch

from mdmm import native, ops, ortho
from test_ortho_gpu import U, check

gpu = pytest.mark.gpu


def test_gradients_are_refused():
    """A matrix that wants a gradient, either way, would lose it."""
    w = torch.ones(4, 4, requires_grad=True)
    with pytest.raises(ValueError, match='gradient'):
        ops.orthogonalise([torch.zeros(4, 4), w])
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match='gradient'):
        ops.orthogonalise([torch.autograd.forward_ad.make_dual(torch.zeros(4, 4), torch.ones(4, 4))])
    for call in (lambda: ops.orthogonalise([w.detach()]), torch.no_grad()(lambda: ops.orthogonalise([w]))):
        with pytest.raises(native.MdmmError):          # (the device's refusal, which comes last)
            call()
