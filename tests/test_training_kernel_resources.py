"""The training operators' kernels keep their working sets in registers.

The cross entropy's epilogue holds 128 sums a thread, the norm's backward pass
its columns of two sums: an array indexed at run time, or an epilogue grown by
one call, would move them to local memory and slow the kernels down without
any change in their results (an out-of-line store routine once cost a third of
the gradients' time). Compiled for sm_100a here, no GPU needed: no kernel may
spill more than a few words.
"""

import pytest

from emeans_b200 import build as ebuild
from tests.test_kernel_resources import _local_memory


@pytest.mark.timeout(900)
@pytest.mark.parametrize("src,kernels", [("linear_ce.cu", ["k_gemm", "k_ce_rows", "k_ce_join"]),
                                         ("linear_ce_small.cu", ["k_ce_small"]),
                                         ("norm.cu", ["k_norm_fwd", "k_norm_bwd"]),
                                         ("adamw.cu", ["k_adamw"])])
def test_training_kernels_spill_at_most_a_few_words(src, kernels):
    try:
        ebuild.nvcc()
    except RuntimeError:
        pytest.skip("nvcc not available")
    found = _local_memory(src)
    for want in kernels:
        assert any(want in k for k in found), (want, sorted(found))
    worst = {k: v for k, v in found.items() if v[0] > 64 or v[1] > 64}
    assert not worst, worst


@pytest.mark.timeout(900)
def test_few_row_kernels_spill_at_most_a_few_words():
    test_training_kernels_spill_at_most_a_few_words("linear_ce_few.cu",
                                                    ["k_few_scores", "k_few_grads"])
