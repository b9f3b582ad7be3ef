"""How many CTAs a row of logits gets, on any number of SMs."""

import itertools

import pytest

from reflex_b200.ops import native


@pytest.mark.parametrize("sms", [16, 20, 63, 64, 132, 148])
def test_sixteen_ctas_only_where_each_has_an_sm_to_itself(sms):
    """More than eight have no room in the form that two CTAs an SM run, which rows get that fill the SMs."""
    for B, V in itertools.product((1, 2, 3, 4, 5, 8, 9, 64, 1500), (1, 4096, 4097, 32003, 151936, 300001, 10 ** 6)):
        C = native.lib().rfx_sample_rows_ctas(B, V, sms)
        assert C in (1, 2, 4, 8) or (C == 16 and B * C <= sms), (B, V, C)


def test_sixteen_for_a_few_wide_rows_of_the_whole_gpu():
    assert [native.lib().rfx_sample_rows_ctas(B, 151936, 148) for B in (1, 4, 5, 64)] == [16, 16, 8, 8]
