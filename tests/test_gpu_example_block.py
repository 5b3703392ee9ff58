"""example_mxfp4_block.py as it is started, on the GPU."""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "comfyui-featherops_amd" / "example_mxfp4_block.py"


@pytest.mark.parametrize("options,halves", [(("--width", "192"), 1), (("--width", "250", "--head-dim", "64"), 1),
                                            (("--width", "192", "--head-dim", "64"), 2)], ids=str)
def test_widths(cuda, options, halves):
    """A width that holds no whole number of heads has the feed-forward half alone."""
    out = subprocess.run([sys.executable, str(EXAMPLE), "--tokens", "40", "--hidden", "320", *options], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert out.stdout.count("MXFP4") == halves and ("no attention half" in out.stdout) == (halves == 1), out.stdout
