"""The SSD needs the C library alone: without the extension module of the operators the package imports, and the operators say
what is missing when they are called."""
import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent.parent / "mamba-ascendc_b200"

PROGRAM = """
import sys
sys.path.insert(0, {package!r})
sys.modules["ascend_kernel._calls"] = None  # an import of it fails
import torch
import ascend_kernel as ak
import ascend_kernel.vmamba2, ascend_kernel.parallel
shape = (1, 128, 2, 64)
try:
    ak.mamba2_ssd_fwd(torch.zeros(shape), *[torch.zeros(1)] * 4, 64)
except RuntimeError as error:
    assert "mamba2_ssd_fwd" in str(error), error
for call in (lambda: ak.rms_norm(torch.zeros(2, 8), torch.ones(8)), lambda: ak.short_conv(torch.zeros(1, 2, 8), torch.ones(8, 4))):
    for _ in range(2):
        try:
            call()
        except ImportError as error:
            assert "_calls.so" in str(error) and "mamba-ascendc_b200/build.py" in str(error), error
        else:
            raise AssertionError("no error")
"""


def test_without_the_extension_module():
    done = subprocess.run([sys.executable, "-c", PROGRAM.format(package=str(PACKAGE))], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
