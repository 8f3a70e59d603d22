"""The Python binding's own checks of verify_draft, verify_sets and linear that need
no GPU: tensors that are not on one."""
import pytest


@pytest.fixture(scope="module")
def hsamp(pkg):
    return pkg.hsamp


def test_tensors_on_the_host_are_refused(hsamp):
    import torch
    x = torch.zeros((2, 8), dtype=torch.bfloat16)
    with pytest.raises(hsamp.HsampError) as e:
        hsamp.linear(x, x)
    assert e.value.status == hsamp.ERR_INVALID
    d, u = torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.float64)
    with pytest.raises(hsamp.HsampError):
        hsamp.verify_draft(torch.zeros((2, 8)), d, u, u, 1)
    with pytest.raises(hsamp.HsampError):
        hsamp.verify_sets(torch.zeros((2, 8), dtype=torch.int32), torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int32), d, u, u, 1)
