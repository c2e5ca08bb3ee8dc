"""What the Python layer refuses before any CUDA call, without a GPU."""
import types

import pytest
import torch

from stadeb200 import kernels as K
from stadeb200 import token_ops as T


@pytest.mark.parametrize("bad,error", [(torch.zeros(1 << 20, dtype=torch.uint8), ValueError),
                                       (torch.zeros(0), ValueError), ([0] * 64, TypeError), (1 << 20, TypeError)])
def test_workspace_must_be_a_tensor_on_the_device(bad, error):
    """The kernels write to it: host memory must not reach them."""
    called, stream = [], types.SimpleNamespace(cuda_stream=0)
    with pytest.raises(error, match="workspace"):
        T._run(lambda *a: called.append(a) or 0, stream=stream, workspace=bad)
    with pytest.raises(error, match="workspace"):
        K._opts(stream, bad)
    assert not called
