"""The serving modules on inputs of another width, which are refused."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import hipgemm_amd as hg
import hipgemm_amd.torch_serving as ts


def test_another_width_is_refused():
    """Twice the features are not twice the rows."""
    lin = ts.W4Linear.from_linear(torch.nn.Linear(64, 40), group_size=32)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, torch.no_grad():
        assert tuple(lin(mode.from_tensor(torch.zeros(4, 64, dtype=torch.bfloat16))).shape) == (4, 40)
        for shape in ((4, 128), (2, 32), (128,), (2, 3, 32)):
            with pytest.raises(hg.HipGemmError):
                lin(mode.from_tensor(torch.zeros(shape, dtype=torch.bfloat16)))
