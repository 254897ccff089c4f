"""Properties of the 8-bit attention kernels' code that no run shows reliably."""
import pytest
from test_attention_build import test_no_path_reads_a_variable_that_was_not_set as no_unset_variable


@pytest.mark.parametrize("source, kernel", [("lw_attn8_decode.hip", "k_attn8_decode")])
def test_no_path_reads_a_variable_that_was_not_set(tmp_path, source, kernel):
    no_unset_variable(tmp_path, source, kernel)
