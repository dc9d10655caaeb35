"""CPU tests of what the serving entry points refuse before anything is launched, beyond test_serving_refusals.py."""
import pytest
import torch

BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _library():
    from vllm_exact import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")


def test_a_workspace_that_is_not_one_run_of_bytes_is_refused():
    """A strided view has other memory between its elements; an expanded one is longer than what it stands on."""
    from vllm_exact import paged_attn as P
    q = torch.zeros(2, 32, 128, dtype=BF)
    need = P.rows_workspace_bytes(2, 32, 128, 5000)
    assert need > 0
    good = torch.empty(need, dtype=torch.uint8)
    assert P._rows_scratch(2, 32, 128, 5000, good, q) == (need, good)
    for bad in (torch.empty(2 * need, dtype=torch.uint8)[::2], torch.empty(1, dtype=torch.uint8).expand(need),
                torch.empty(need // 4 + 1, 2, dtype=torch.float32).t()):
        with pytest.raises(ValueError, match="contiguous"):
            P._rows_scratch(2, 32, 128, 5000, bad, q)
        with pytest.raises(ValueError, match="contiguous"):  # the same of a call that needs none of it
            P._rows_scratch(2, 32, 128, 1, bad, q)
    got, fresh = P._rows_scratch(2, 32, 128, 5000, torch.empty(10, dtype=torch.uint8), q)  # too small: one is made
    assert got == need and fresh.numel() == need
