"""The largest and least scales that the attention entries take, before anything is launched: no GPU needed."""
import pytest

from fuel_b200 import _lib as L

F32, F16, BF16 = 0, 1, 30
A = 4096   # an aligned address that nothing is read from: every call below is refused or has no rows


def decode(act, scale, seqs):
    return L.lib.fuelq_paged_attn_decode(act, act, A, 4096, A, A, A, A, A, seqs, 32, 8, 128, 16, 8, 2, scale, A, 1 << 40, None)


def prompt(act, scale, rows):
    return L.lib.fuelq_prompt_attn(act, A, 4096, A, 1024, A, 1024, A, A, 4, rows, 32, 8, 128, scale, A, 1 << 40, None)


@pytest.mark.parametrize("call", [decode, prompt])
@pytest.mark.parametrize("act", [F32, F16, BF16])
def test_scales_that_pass_f32_with_log2_e(call, act):
    """Scores are powers of two on the way, scale * log2(e) of them: an infinite factor would make NaN of a score of zero."""
    assert call(act, 2.0 ** 127, 0) == L.OK
    for scale in (1.001 * 2.0 ** 127, 2.4e38, 3.4e38):
        assert call(act, scale, 0) == L.INVALID_PROBLEM and call(act, scale, 4) == L.INVALID_PROBLEM


@pytest.mark.parametrize("call", [decode, prompt])
@pytest.mark.parametrize("act", [F32, F16, BF16])
def test_scales_that_leave_a_factor_no_bits(call, act):
    """Below 2^-100 the product with a row's power of two would lose its bits before the keys' powers bring it back."""
    assert call(act, 2.0 ** -100, 0) == L.OK
    for scale in (0.99 * 2.0 ** -100, 2.0 ** -126, 1e-44):
        assert call(act, scale, 0) == L.INVALID_PROBLEM and call(act, scale, 4) == L.INVALID_PROBLEM
