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


@pytest.mark.parametrize("u_draw", [None, "scalar"])
@pytest.mark.parametrize("draft", ["vector", "scalar"])
def test_missing_and_scalar_vectors_are_refused(hsamp, u_draw, draft):
    """(on the host: the checks that verify_draft and verify_sets share)"""
    import torch
    d = torch.zeros(() if draft == "scalar" else 1, dtype=torch.int32)
    v = None if u_draw is None else torch.zeros((), dtype=torch.float64)
    with pytest.raises(hsamp.HsampError) as e:
        hsamp._seq_args(hsamp.Draft(), "verify_draft", torch.device("cpu"), d, torch.zeros(1, dtype=torch.float64), v, 1, None,
                        None, None, True, None)
    assert e.value.status == hsamp.ERR_INVALID
    with pytest.raises(hsamp.HsampError):
        hsamp._seq_args(hsamp.Draft(), "verify_draft", torch.device("cpu"), torch.zeros((), dtype=torch.int32),
                        torch.zeros(1, dtype=torch.float64), torch.zeros(1, dtype=torch.float64), 1, None, None, None, True, None)
