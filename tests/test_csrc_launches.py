"""Every dependent launch names its kernel, so that the rules on the kernels' text reach all of them."""
import glob
import os

from test_csrc_rules import CSRC, _dependent, _kernels, _source


def test_dependent_launches_name_kernels_of_their_file():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = _source(path)
        assert _dependent(text) <= set(_kernels(text)), (os.path.basename(path), _dependent(text) - set(_kernels(text)))
