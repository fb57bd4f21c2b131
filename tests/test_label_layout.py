"""Where label operators' scratch memory and codes lie, on the CPU: strides that vector loads need, and offsets that pass 32 bits."""
import pytest

from renee_amd._lib import lib


@pytest.mark.parametrize("rows", [1, 3, 256, 300])
@pytest.mark.parametrize("K", [9, 300, 6000])
def test_maxima_beside_logits_are_rows_of_whole_pieces(rows, K):
    """The selection reads a row's maxima, one half for every 32 labels, in pieces of 16 bytes: each row begins on one, and the last row's
    last piece is inside the workspace."""
    h = lib()
    for L in [*range(65_473, 65_900, 7), 70_001, 131_072, 320_001, 414_001, 1_310_720, 2_812_281, (1 << 30) - 1]:
        if L < K * 64:
            continue
        d = 4096  # wide enough for every K to go by logits
        logits = (rows * -(-L // 64) * 64 * 2 + 15) // 16 * 16
        maxima = h.xfc_mx4_topk_workspace_bytes(rows, L, d, K) - logits
        blocks = -(-L // 32)
        if rows >= 32 and maxima < 0:  # by maxima alone
            continue
        if maxima == 0:  # too few blocks for them to be of use
            assert blocks < 2048 or blocks < 2 * K
            continue
        assert maxima % rows == 0 and maxima // rows % 16 == 0
        assert maxima // rows >= -(-blocks // 8) * 16
