"""What no run on a CPU and no passing run on a GPU can show of the kernels of libta_nn.so, read from their sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transferattack_amd", "csrc", "nn")


def test_lds_written_by_one_lane_is_ordered_before_it_is_read():
    """distil_rows: lane 0 writes `side`, the whole first wave reads it; with one wave to a workgroup block_max and block_sum have no
    barrier, so the order has to be asked for right behind the write"""
    text = open(os.path.join(CSRC, "distil.hip")).read()
    writes = [m.end() for m in re.finditer(r"if \(tid == 0\) side = t;", text)]
    assert len(writes) == 1
    assert re.match(r"\s*(wave_lds_order|__syncthreads)\(\);", text[writes[0]:])
