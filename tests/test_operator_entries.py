"""What the C entries of linear and latent attention refuse beside what their own tests list."""
import pytest

from flashkda_b200 import _lib
from test_latent_attention import decode_params, prompt_params
from test_linear_attention import params


@pytest.mark.parametrize("over", [dict(cu_seqlens=0x1004), dict(cu_seqlens=0x1001)])
def test_cumulative_lengths_off_their_alignment_are_refused(over):
    """A kernel would read them as 64-bit numbers at an address that is none of such a number."""
    assert _lib.lib().fkda_linear_attention_fwd(params(**over), None) == 8
    assert _lib.lib().fkda_latent_attention_fwd(prompt_params(cu_seqlens_k=0x1000, **over), None) == 8
    assert _lib.lib().fkda_latent_attention_fwd(prompt_params(cu_seqlens=0x1000, cu_seqlens_k=over["cu_seqlens"]), None) == 8


@pytest.mark.parametrize("scale", [1e-40, -1e-40, 1.1754942e-38, 3e38])
def test_softmax_scales_that_become_nothing_or_infinite_are_refused(scale):
    """Scale times log2(e) would be flushed to 0, or overflow, and 0 or infinity times a masked or a zero score is no number."""
    assert _lib.lib().fkda_latent_attention_fwd(prompt_params(scale=scale), None) == 11
    assert _lib.lib().fkda_latent_attention_decode(decode_params(scale=scale), None) == 11
