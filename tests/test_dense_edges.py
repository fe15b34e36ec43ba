"""The dense feed-forward operators at their edges, without a GPU: waits that the source has to ask for, sizes that few launches hold, refusals."""
import os
import re

from tests import support

CSRC = os.path.join(support.ROOT, "numkong_amd", "csrc")


def test_tiles_wait_for_every_load_into_lds_before_they_put_sums_there():
    """Behind the loop over the stages loads into LDS (zeros, of stages past the end) are still on their way, into arrays that another wavefront puts
    its sums into: each wavefront has to wait for its own before they meet. A barrier alone does not, by contract."""
    source = open(os.path.join(CSRC, "dense_tiles_gfx950.hpp")).read()
    wait = re.search(r"void arrive_and_meet\(\) \{(.*?)\n\}", source, flags=re.S).group(1)
    assert re.search(r"s_waitcnt\(0x0070\).*s_barrier\(\)", wait, flags=re.S)  # vmcnt(0) and lgkmcnt(0), then the barrier
    kernel = source[source.index("void tile_kernel("):]
    behind = kernel[kernel.index("stage(a1, b1, a0, b0, s + 1"):]
    before_sums = re.sub(r"//.*", "", behind[:behind.index("float *const room")])
    assert "arrive_and_meet();" in before_sums and "__syncthreads" not in before_sums and "s_barrier" not in before_sums
