"""What the modules around the layers take and refuse, as far as it needs no GPU."""
import pytest
import torch


def test_a_checkpoint_off_the_gpu_is_not_decoded():
    import sparse
    kept = sparse.ActivationCheckpoint(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8), (4, 64), torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kept.decode()
