"""Refusals of the paged operators at the edges of their ranges, without a GPU."""

from cs348k_fast_attention_grammar_b200 import _lib
from test_paged_cpu import ATTN, P, _codes


def test_scales_beyond_fp32():
    """The kernels scale in fp32, times log2(e): what is infinite there is refused."""
    lib, code = _lib.load(), _codes()
    for scale in (3e38, -3e38, 1e300, -1e300, float("inf"), float("nan")):
        args = ATTN.pack(*(P,) * 7, 0, 3, 3, 4, 2, 64, 4, 16, 2, 2, 256, 64, 256, 64,
                         *(2048, 128, 64) * 2, 1, 1, scale)
        assert lib.fa_paged_attn(args, P, 1 << 40, None) == code["FA_ERR_ARG"], scale
        assert lib.fa_paged_attn_workspace(args) == -code["FA_ERR_ARG"], scale
