"""Gated feed-forward block and residual norms: size queries and refusals that
need no GPU (the library checks its arguments before any CUDA call on them;
the Python surface checks its tensors before the library)."""
import ctypes as C

import pytest
import torch

from mogecpp_b200 import lib as L
from mogecpp_b200.sparse import SparseCudaExecutor


def test_workspace_queries():
    lib = L.load()
    # the hidden values in 16 bits, then the K split's partial sums where few rows leave SMs idle
    assert lib.msc_gated_ffn_workspace_bytes(100000, 256, 512) == 100000 * 512 * 2
    # one kernel keeps them on the SM where the channels are few and the rows many
    assert lib.msc_gated_ffn_workspace_bytes(100000, 128, 512) == 0
    assert lib.msc_gated_ffn_workspace_bytes(1, 1024, 4096) >= 4096 * 2
    assert lib.msc_gated_ffn_workspace_bytes(0, 128, 512) >= 0
    for bad in ((-1, 128, 512), (1, 0, 512), (1, 128, 0), (1, 8200, 512), (1, 128, 65544), (1 << 40, 128, 512)):
        assert lib.msc_gated_ffn_workspace_bytes(*bad) == 0
        assert lib.msc_gated_ffn_backward_workspace_bytes(*bad) == 0
        assert lib.msc_ffn_stack_workspace_bytes(*bad) == 0
    # dg, du and h
    assert lib.msc_gated_ffn_backward_workspace_bytes(100000, 128, 512) >= 3 * 100000 * 512 * 2
    # two row buffers and the block's own
    assert lib.msc_ffn_stack_workspace_bytes(1000, 128, 512) == (
        2 * 1000 * 128 * 2 + lib.msc_gated_ffn_workspace_bytes(1000, 128, 512))
    for n, c, ns in ((1, 8, 0), (400000, 128, 2), (400000, 128, 127), (1000, 8192, 1 << 15)):
        b = lib.msc_residual_norm_backward_workspace_bytes(n, c, ns)
        assert b >= (4 + max(ns, 1)) * c * 4
        # the slabs of all units stay within 64 MiB unless one alone is larger
        assert b <= max(64 << 20, (4 + max(ns, 1)) * c * 4 + 256)
    assert lib.msc_residual_norm_backward_workspace_bytes(-1, 128, 0) == 0
    assert lib.msc_residual_norm_backward_workspace_bytes(1, 8200, 0) == 0
    assert lib.msc_residual_norm_backward_workspace_bytes(1, 128, -1) == 0
    assert lib.msc_residual_norm_backward_workspace_bytes(1, 128, (1 << 15) + 1) == 0


def test_sizes_grow_with_rows():
    lib = L.load()
    for q in (lib.msc_gated_ffn_workspace_bytes, lib.msc_gated_ffn_backward_workspace_bytes):
        assert q(2000000, 256, 512) > q(1000000, 256, 512) > q(100000, 256, 512) > 0
        # past 32 bits
        assert q(70000000, 256, 512) > 1 << 32


def test_null_context_is_refused():
    lib = L.load()
    assert lib.msc_gated_ffn(None, None, 0, 0, None, None, None, 0, None) == -1
    assert lib.msc_gated_ffn_backward(None, None, 0, 0, None, None, None, None, 0, None) == -1
    assert lib.msc_residual_norm(None, None, 0, None, None, None, None, None, None) == -1
    assert lib.msc_residual_norm_backward(None, None, 0, None, None, None, None, None, None, None, 0, None) == -1
    assert lib.msc_ffn_stack(None, None, 0, 0, 0, None, 0, 0, None, None, 0, None) == -1
    assert "context" in lib.msc_last_error().decode()


def test_struct_sizes_match_the_header(tmp_path):
    """The ctypes structures and the C header agree on every size."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    if shutil.which("gcc") is None:
        pytest.skip("gcc is not installed")
    pairs = {"msc_norm": L.Norm, "msc_residual_norm_desc": L.ResidualNormDesc,
             "msc_residual_norm_grads": L.ResidualNormGrads, "msc_ffn": L.Ffn, "msc_ffn_grads": L.FfnGrads,
             "msc_ffn_block": L.FfnBlock}
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "moge_sparse_cuda.h"\nint main(void) {\n' + "".join(
        f'printf("{k} %lu\\n", (unsigned long)sizeof({k}));\n' for k in pairs) + "return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for k, t in pairs.items():
        assert int(out[k]) == C.sizeof(t), k


class _NoLibrary:
    """Stands in for the library: any call through it fails the test."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture
def host_ex():
    ex = SparseCudaExecutor.__new__(SparseCudaExecutor)
    ex.device, ex.ctx, ex.lib = 0, None, _NoLibrary()
    return ex


def test_host_tensors_are_refused(host_ex):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    ffn = dict(w_gate=torch.zeros(128, 64, dtype=torch.bfloat16), w_up=torch.zeros(128, 64, dtype=torch.bfloat16),
               w_down=torch.zeros(64, 128, dtype=torch.bfloat16))
    for call in (lambda: host_ex.gated_ffn(x, ffn), lambda: host_ex.gated_ffn_backward(x, x, ffn),
                 lambda: host_ex.residual_norm(x, x), lambda: host_ex.residual_norm_backward(x, x, x, None),
                 lambda: host_ex.ffn_stack(x, [dict(ffn=ffn)])):
        with pytest.raises(L.MscError, match="cuda:0"):
            call()
