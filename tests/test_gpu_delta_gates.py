"""Gates of the delta rule in every layout that a caller may have them in."""
import numpy as np
import pytest
import torch

from tests._decode import Delta, same
from vllm_sly_radiance_amd import _native_decode
from vllm_sly_radiance_amd import radiance_gdn as G

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(gpu_lib):
    return _native_decode.lib()


LAYOUTS = {
    "one number a token for all heads": lambda x: x[:, :1].expand(-1, x.shape[1]),
    "one row of numbers for all tokens": lambda x: x[:1].expand(x.shape[0], -1),
    "one number": lambda x: x[:1, :1].expand(x.shape),
    "every other column": lambda x: torch.cat([x, x], 1)[:, ::2],
    "heads first": lambda x: x.T.contiguous().T,
}


@pytest.mark.parametrize("layout", LAYOUTS.values(), ids=LAYOUTS.keys())
@pytest.mark.parametrize("lens", [[1], [3, 2], [40, 90]], ids=str)
def test_layouts_of_gates(lens, layout):
    """The values are those of a copy, whatever the strides; a view's own elements are all there is of it."""
    for which in (3, 4):
        d = Delta(np.random.default_rng(31), lens, (2, 4, 128, 64))
        args, plain = d.device(), d.device()
        args[which] = layout(args[which].clone())
        plain[which] = args[which].contiguous()
        assert torch.equal(G.gated_delta_rule(*args), G.gated_delta_rule(*plain)) and same(args[7], plain[7])
