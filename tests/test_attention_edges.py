"""-m "not gpu": corners of the attention-layer operators through the SIMT emulator; the checks themselves are in tests/attention_edges.py."""
import pytest
import torch

import attention_edges as ae

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_key_rows_that_share_memory(emu_lib, dt, bad):
    ae.check_shared_key_rows(emu_lib, "cpu", dt, bad)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_unturned_elements(emu_lib, dt, adjacent, norm):
    ae.check_unturned_elements(emu_lib, "cpu", dt, adjacent, norm)
