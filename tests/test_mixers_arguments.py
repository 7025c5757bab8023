"""What is no device tensor is refused by name, whatever it is."""
import numpy as np
import pytest
import torch

from fable5_llm_amd import mixers


class Ctx:
    h, device = None, 0


@pytest.mark.parametrize("bad", [None, 3, np.zeros((2, 1, 64), np.float32), torch.zeros(2, 1, 64)])
@pytest.mark.parametrize("name", ["q", "k", "v", "out", "g", "beta", "state"])
def test_delta_rule(bad, name):
    class OnDevice:                                   # as much of a tensor as is looked at first
        is_cuda, dtype, shape = True, torch.float32, torch.Size((2, 1, 64))

        def get_device(self):
            return 0

        def dim(self):
            return 3

    d = {n: OnDevice() for n in ("q", "k", "v", "g", "beta", "state", "out")}
    d[name] = bad
    with pytest.raises(ValueError, match=f"^{name}: must be a device tensor"):
        mixers.delta_args(Ctx, **d, cu=None, ws=None, slots=None, scale=None, norm=True, eps=1e-6,
                          fresh=False, frac=0, out_frac=0)
