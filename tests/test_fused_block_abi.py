"""Arguments that the layer norm and linear entry points refuse, and their workspace sizes, on the host: every check
comes before the first use of the GPU."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

P = ctypes.c_void_p(256)         # stands for a device pointer; never read


@pytest.fixture(scope="module")
def lib():
    from aimet_amd._lib import lib as l
    return l


def _refused(lib, rc, word):
    assert rc == -1, rc
    assert word.encode() in lib.miq_last_error(), lib.miq_last_error()


@pytest.mark.parametrize("suffix", ["f32", "bf16"])
def test_layer_norm_refusals(lib, suffix):
    fwd, bwd = getattr(lib, "miq_layer_norm_fwd_" + suffix), getattr(lib, "miq_layer_norm_bwd_" + suffix)
    _refused(lib, fwd(P, None, None, -1, 8, 1e-5, P, None, None, None), "rows")
    _refused(lib, fwd(P, None, None, 4, 0, 1e-5, P, None, None, None), "width")
    _refused(lib, fwd(P, None, None, 1 << 31, 8, 1e-5, P, None, None, None), "2^31")
    _refused(lib, fwd(None, None, None, 4, 8, 1e-5, P, None, None, None), "null")
    _refused(lib, fwd(P, None, None, 4, 8, 1e-5, None, None, None, None), "null")
    _refused(lib, fwd(P, None, None, 4, 8, 1e-5, P, P, None, None), "together")
    _refused(lib, bwd(P, P, None, None, P, 4, 8, P, None, None, None, None), "null")
    _refused(lib, bwd(P, P, None, P, P, 4, 8, P, P, None, None, None), "workspace")
    assert fwd(None, None, None, 0, 8, 1e-5, None, None, None, None) == 0
    assert bwd(None, None, None, None, None, 0, 8, None, None, None, None, None) == 0
    assert lib.miq_layer_norm_bwd_workspace_bytes(-1, 8) == 0
    assert lib.miq_layer_norm_bwd_workspace_bytes(1000, 64) > 0


@pytest.mark.parametrize("suffix", ["f32", "bf16"])
def test_linear_refusals(lib, suffix):
    fwd, bwd = getattr(lib, "miq_linear_fwd_" + suffix), getattr(lib, "miq_linear_bwd_" + suffix)
    big = 1 << 40
    _refused(lib, fwd(P, P, None, None, -1, 8, 8, 0, P, None, P, big, None), "negative")
    _refused(lib, fwd(P, P, None, None, 1 << 31, 8, 8, 0, P, None, P, big, None), "2^31")
    _refused(lib, fwd(P, P, None, None, 4, (1 << 27) + 1, 8, 0, P, None, P, big, None), "2^27")
    _refused(lib, fwd(P, P, None, None, 4, 8, (1 << 27) + 1, 0, P, None, P, big, None), "2^27")
    _refused(lib, fwd(P, P, None, None, 4, 8, 8, 5, P, None, P, big, None), "activation")
    _refused(lib, fwd(None, P, None, None, 4, 8, 8, 0, P, None, P, big, None), "null")
    _refused(lib, fwd(P, P, None, None, 4, 8, 8, 0, None, None, P, big, None), "null")
    _refused(lib, bwd(P, None, P, P, 4, 8, 8, 3, P, P, P, P, big, None), "null")            # saved is missing
    _refused(lib, bwd(P, None, None, P, 4, 8, 8, 0, P, P, P, P, big, None), "x")
    _refused(lib, bwd(P, None, P, None, 4, 8, 8, 0, P, P, P, P, big, None), "weight")
    _refused(lib, bwd(P, P, P, P, 4, 8, 8, 3, P, P, P, P, 0, None), "workspace")
    for rows, n_in, n_out in ((1, 64, 64), (300, 1000, 77), (5000, 512, 4096)):
        need = lib.miq_linear_workspace_bytes(rows, n_in, n_out, 3, int(suffix == "bf16"), 0, 1)
        if need:
            _refused(lib, fwd(P, P, None, None, rows, n_in, n_out, 3, P, None, P, need - 1, None), "workspace")
    assert fwd(None, None, None, None, 0, 8, 8, 0, None, None, None, 0, None) == 0
    assert lib.miq_linear_workspace_bytes(-1, 8, 8, 0, 0, 1, 1) == 0


def test_linear_workspace_of_layers_without_outputs():
    """In a process of its own: a division by zero on the host would end the test run, not fail a test."""
    code = ("import sys; sys.path.insert(0, %r)\n"
            "from aimet_amd._lib import lib\n"
            "for bf16 in (0, 1):\n"
            "    for activation in (0, 3):\n"
            "        for shape in ((5, 24, 0), (300, 4096, 0), (0, 24, 0), (5, 0, 0), (5, 0, 7), (0, 0, 0)):\n"
            "            for backward in (0, 1):\n"
            "                for aligned in (0, 1):\n"
            "                    print(bf16, activation, shape, backward, aligned, end=' ', flush=True)\n"
            "                    print(lib.miq_linear_workspace_bytes(*shape, activation, bf16, backward, aligned))"
            % ROOT)
    run = subprocess.run([sys.executable, "-c", code], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, check=False)
    lines = run.stdout.splitlines()
    assert run.returncode == 0, (run.returncode, lines[-1:], run.stderr)
    assert len(lines) == 96 and all(int(line.split()[-1]) >= 0 for line in lines)


@pytest.mark.parametrize("rows", [(1 << 27) + 1, 160_000_000, (1 << 31) - 1])
@pytest.mark.parametrize("features", [8, 16, 64])
def test_sums_over_more_rows_than_a_row_of_halves_holds(lib, rows, features):
    """The weight's gradient sums over the rows.  Rows of halves that long are past what a lane's 32-bit offset spans; the
    way without halves needs no copy of x, which shows in the workspace: halves of x take 4 bytes for each value."""
    assert 0 < lib.miq_linear_workspace_bytes(rows, features, features, 0, 0, 1, 1) < rows * features * 4


def test_functions_refuse_before_any_launch():
    import torch
    from aimet_amd.v2.nn import fused
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call in (lambda: fused.linear(x, w), lambda: fused.layer_norm(x, 8), lambda: fused.layer_norm(x, 7),
                 lambda: fused.layer_norm(x, ()), lambda: fused.layer_norm(x, 8, torch.ones(7))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        fused.linear(x, w, None, "swish")
    with pytest.raises(ValueError):
        fused.FusedLinear(8, 6, activation="swish")
    with pytest.raises(ValueError):
        fused.FusedLinear.from_linear(torch.nn.Linear(8, 6), "swish")


def test_only_the_functions_of_the_torch_binding_need_it(tmp_path):
    """A tree without _native.so: the package imports and quantizes, layer_norm() and linear() say what is missing."""
    package = tmp_path / "aimet_amd"
    shutil.copytree(os.path.join(ROOT, "aimet_amd"), package,
                    ignore=shutil.ignore_patterns("*.so", "*.o", "__pycache__", "csrc"))
    os.symlink(os.path.join(ROOT, "aimet_amd", "libmiq.so"), package / "libmiq.so")
    code = ("import sys; sys.path.insert(0, %r)\n"
            "from aimet_amd import _lib\n"
            "assert _lib.__file__.startswith(%r) and _lib.lib.miq_version() >= 1\n"
            "import aimet_amd.common.libpymo as pymo\n"
            "assert 'torch' not in sys.modules\n"
            "import torch, aimet_amd.v1.quantsim, aimet_amd.v2.quantsim\n"
            "from aimet_amd.v2.nn import fused\n"
            "fused.FusedLinear(8, 6)\n"
            "for call in (lambda: fused.linear(torch.zeros(4, 8), torch.zeros(6, 8)),\n"
            "             lambda: fused.layer_norm(torch.zeros(4, 8), 8)):\n"
            "    try:\n"
            "        call()\n"
            "    except ImportError as e:\n"
            "        assert '_native.so' in str(e)\n"
            "    else:\n"
            "        raise AssertionError('not refused')\n" % (str(tmp_path), str(tmp_path)))
    run = subprocess.run([sys.executable, "-c", code], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, check=False,
                         cwd=str(tmp_path))
    assert run.returncode == 0, run.stderr
