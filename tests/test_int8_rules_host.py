"""Which 8-bit transforms need scratch memory, which tells the kernel that takes them apart."""
import pytest

from gnn_cuda_b200 import _native as N

ALIGNED = 1 << 20


def _bytes(x_type, m, k, n=512):
    pitch = (k + 15) // 16 * 16
    return N.lib().gnn_linear_int8_workspace_bytes(ALIGNED, x_type, k if x_type == N.GNN_ROWS_FP32 else pitch, ALIGNED,
                                                   pitch, N.GNN_ROWS_FP32, m, k, n)


@pytest.mark.parametrize("m,k,few", [(1, 1, True), (1, 2048, True), (1, 2049, False), (1, 4096, False), (1, 40960, False),
                                     (2, 2048, True), (2, 4096, False), (16, 512, True), (16, 513, False), (17, 64, False)])
def test_long_fp32_rows_are_quantised_by_the_whole_device(m, k, few):
    """The few-rows kernel quantises a row with one warp of every block; a long row goes to the quantiser."""
    assert (_bytes(N.GNN_ROWS_FP32, m, k) == 0) == few


@pytest.mark.parametrize("m,k", [(1, 40960), (2, 4096), (16, 513)])
def test_8_bit_rows_need_no_scratch(m, k):
    assert _bytes(N.GNN_ROWS_INT8, m, k) == 0
