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


@pytest.mark.parametrize("n", [1, 4, 5, 8, 9, 64, 128, 300, 1237, 4736, 18943, 18944])
@pytest.mark.parametrize("c", [8, 64, 128, 256, 512, 1024, 8192])
def test_stack_workspace_covers_smaller_blocks(n, c):
    """A stack's workspace is asked for with the largest hidden size: it holds
    every smaller block's, though a block of its own may need less as it grows
    (fewer K splits, or another path)."""
    lib = L.load()
    rows = 2 * ((n * c * 2 + 255) // 256 * 256)
    most = 0
    for hidden in [*range(8, 4200, 8), *range(4200, 65536, 1000), 65536]:
        most = max(most, rows + lib.msc_gated_ffn_workspace_bytes(n, c, hidden))
        assert lib.msc_ffn_stack_workspace_bytes(n, c, hidden) >= most, hidden
    # around the end of the dot products (8 rows of 128 channels: 16,384 hidden units)
    size = [lib.msc_ffn_stack_workspace_bytes(n, c, h) for h in range(8, 65537, 8)]
    assert all(a <= b for a, b in zip(size, size[1:]))
    # no more than the splits' own rounding costs
    assert size[-1] <= 2 * most


def test_wrong_arguments_are_refused_as_such(host_ex):
    """Missing weights, weights and gates of another rank or kind, an unknown
    branch type: the library's own error, before the library."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    f32 = x.float()
    w, d = torch.zeros(128, 64, dtype=torch.bfloat16), torch.zeros(64, 128, dtype=torch.bfloat16)
    ffn = dict(w_gate=w, w_up=w, w_down=d)
    bad = [{**ffn, "w_gate": w[0]}, {**ffn, "w_down": None}, {"w_gate": w, "w_up": w}, {**ffn, "w_up": 1.0},
           {**ffn, "w_gate": torch.zeros((), dtype=torch.bfloat16)}, {}]
    for f in bad:
        for call in (lambda: host_ex.gated_ffn(x, f), lambda: host_ex.gated_ffn_backward(x, x, f),
                     lambda: host_ex.ffn_stack(f32, [dict(ffn=f)])):
            with pytest.raises(L.MscError, match="w_"):
                call()
    for gate in (torch.zeros(()), torch.zeros(1, 1, 64), torch.zeros(8, 64).t(), 0.5):
        with pytest.raises(L.MscError, match="gate"):
            host_ex.residual_norm(f32, f32, gate=gate, coords=torch.zeros(4, 4, dtype=torch.int32))
        with pytest.raises(L.MscError, match="gate"):
            host_ex.residual_norm_backward(f32, f32, f32, None, gate=gate, coords=torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(L.MscError, match="branch"):
        host_ex.residual_norm(f32, pre=dict(kind="rms"), branch_dtype=torch.float64)
