"""Feed-forward blocks and residual norms: empty inputs and size queries, on
the host alone."""
import pytest
import torch

from mogecpp_b200 import lib as L
from mogecpp_b200.sparse import SparseCudaExecutor
from test_ffn_host import _NoLibrary


@pytest.fixture
def host_ex():
    """Checks host tensors as its own (their device index is -1) and fails
    when a call gets past the checks."""
    ex = SparseCudaExecutor.__new__(SparseCudaExecutor)
    ex.device, ex.ctx, ex.lib = -1, None, _NoLibrary()
    return ex


def test_gate_of_no_samples_is_refused(host_ex):
    """A [0, c] gate has address zero and no samples, which the library reads
    as no gate at all: the branch would be added as it is."""
    x = torch.zeros(4, 64)
    gate, coords = torch.zeros(0, 64), torch.zeros(4, 4, dtype=torch.int32)
    ffn = dict(w_gate=torch.zeros(128, 64, dtype=torch.bfloat16), w_up=torch.zeros(128, 64, dtype=torch.bfloat16),
               w_down=torch.zeros(64, 128, dtype=torch.bfloat16))
    for call in (lambda: host_ex.residual_norm(x, x, gate=gate, coords=coords),
                 lambda: host_ex.residual_norm_backward(x, x, x, None, gate=gate, coords=coords),
                 lambda: host_ex.ffn_stack(x, [dict(ffn=ffn, gate=gate)], coords=coords)):
        with pytest.raises(L.MscError, match="at least one sample"):
            call()
