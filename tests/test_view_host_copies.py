"""Host copies of views by element type (the views lie over CPU tensors here: the copies are torch's)."""
import numpy as np
import pytest
import torch

import momiru_b200 as mb


def test_integers_keep_their_values():
    v = mb.DeviceView.from_torch(torch.zeros(6, dtype=torch.int32))
    ids = np.array([0, -1, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31), 123456789], np.int32)
    v.copy_from_host(ids)
    assert np.array_equal(v.to_host(), ids) and v.to_host().dtype == np.int32
    v.copy_from_host(ids[::-1].astype(np.int64))
    assert np.array_equal(v.to_host(), ids[::-1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_floats_round_once(dtype):
    v = mb.DeviceView.from_torch(torch.zeros(2, 3, dtype=dtype)).transpose()
    x = np.random.default_rng(0).standard_normal((3, 2)).astype(np.float32)
    v.copy_from_host(x)
    assert np.array_equal(v.to_host(), torch.from_numpy(x).to(dtype).float().numpy())
