"""How much one launch of the attention side takes, on a host-only context."""
import pytest

import moe_rocm as M

X = 0x1000  # any non-NULL address: a host-only context never follows it


@pytest.fixture
def hctx():
    ctx = M.Context(M.DEVICE_NONE)
    yield ctx
    ctx.close()


OK, TOO_MANY = M.MR_E_NODEV, M.MR_E_INVAL  # a host-only context refuses what fits a launch for want of a device


@pytest.mark.parametrize("rows,heads,seqs,status", [
    (128 * (2 ** 24 - 10), 1, 1, OK), (128 * (2 ** 24 - 9), 1, 1, TOO_MANY), (128 * (2 ** 24 - 4), 1, 1, TOO_MANY),
    (128 * (2 ** 20 - 3), 16, 1, OK), (128 * (2 ** 20 - 3), 16, 2, TOO_MANY), (128, 8, 2 ** 21 - 3, OK),
    (128, 5, 3355439, OK), (128, 5, 3355440, TOO_MANY)])
def test_tiles_of_a_prompt_fit_a_launch(hctx, rows, heads, seqs, status):
    """(rows / 128 + sequences + 1) heads tiles, launched in eights of 256 threads, less than 2^32 threads in all."""
    q = M.Heads(X, heads, M.F16)
    with pytest.raises(M.MoeRocmError) as ei:
        M.attn_prefill(hctx, 64, q, q, q, rows, rows, seqs, X, X, q)
    assert ei.value.status == status, ei.value.message
