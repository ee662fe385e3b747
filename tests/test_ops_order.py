"""Order of shared-memory accesses in the serving operators' kernels that the
emulator, whose memory is sequentially consistent, cannot show."""
import os
import re

from simt_lib import CSRC


def test_cursor_writes_are_ordered_before_the_lanes_read_them():
    """Lane 0 moves a warp's cursor in shared memory and every lane reads it
    behind the call: a __syncwarp has to stand between the two, since a shuffle
    orders no memory.  Before the write, too, where lanes read the cursor's
    old place (all calls but the first)."""
    src = open(os.path.join(CSRC, "l3g_chunk_attn.cuh")).read()
    for name, older_reads in (("first", False), ("next", True)):
        body = re.search(r"auto %s = \[&\] \{(.*?)\n  \};" % name, src, re.S).group(1)
        write = body.index("if (lane == 0) more = chunk_%s<BN>(a, sh, c);" % name)
        syncs = [m.start() for m in re.finditer(r"__syncwarp\(\);", body)]
        assert any(write < s < body.index("__shfl_sync") for s in syncs), name
        assert not older_reads or any(s < write for s in syncs), name
