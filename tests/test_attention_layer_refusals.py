"""What MultiHeadAttention.attend refuses before anything is launched (no GPU needed)."""
import pytest
import torch

from ttdg_mgm_amd.GModule.utils.attentions import MultiHeadAttention


def test_heads_that_do_not_divide_the_channels():
    """6 heads of 16 channels each are 96 of 100: the output projection has no place for them."""
    m, x = MultiHeadAttention(100, 6), torch.zeros(2, 3, 100)
    with pytest.raises(ValueError, match="6 heads"):
        m.attend(x, x)
