"""A wait that runs out in attention over a paged cache can be read by who makes the call through the extension (no GPU)."""
import pytest
import torch


def test_the_status_is_a_call_of_its_own(ext, capi):
    assert "l3ci_paged_attention_poll" in capi.EXPORTS
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ext.paged_attention_status(torch.zeros(1))
