"""The cross entropy's kernels that hand registers from one warpgroup to the
others (setmaxnreg) are launched with what the shares add up to.

The shares are 128 threads of 72 and 256 of 216, together the 384 of 168 that a
block may be launched with. A build that took fewer would leave the larger share
waiting for registers that never come, so every such kernel has to report 168.
Compiled for sm_100a here, no GPU needed."""

import os
import re

import pytest

from emeans_b200 import build as ebuild
from tests.test_kernel_resources import _ptxas_report


@pytest.mark.timeout(900)
def test_kernels_that_share_registers_are_launched_with_all_of_them():
    try:
        ebuild.nvcc()
    except RuntimeError:
        pytest.skip("nvcc not available")
    src = open(os.path.join(ebuild.CSRC, "linear_ce.cu")).read()
    less, more = (int(re.search(r"setmaxnreg\.%s\.sync\.aligned\.u32 (\d+)" % w, src).group(1))
                  for w in ("dec", "inc"))
    each = (128 * less + 256 * more) // 384
    assert (each, (128 * less + 256 * more) % 384) == (168, 0)
    found = re.findall(r"Compiling entry function '(\S*k_gemm\S*)'.*?Used (\d+) registers",
                       _ptxas_report("linear_ce.cu"), re.S)
    # k_gemm<epilogue, CTAs, terms, width, chained, fine>
    chained = [(name, int(regs)) for name, regs in found
               if re.search(r"k_gemmILi\dELi\dELb[01]ELi\d+ELb1ELb[01]E", name)]
    assert len(found) >= 20 and len(chained) >= 10, [n for n, _ in found]
    assert all(regs == each for _, regs in chained), chained
