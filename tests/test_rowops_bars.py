"""The comparisons of the long gradients see a lost piece (on the host: the mistakes are planted in the expected sums)."""
import numpy as np
import pytest

from test_gpu_rowops import WHOLE, whole_case


@pytest.mark.parametrize("n,rows,d,how", WHOLE)
def test_a_lost_piece_is_seen(n, rows, d, how):
    """The sorted tokens are added in chunks of 16, 64 or 256, and a long row's chunks in eighths: without one chunk, without one
    eighth of the longest row, and without one token the sums differ in every column."""
    grad, ids, sums = whole_case(n, rows, d, how)
    key = np.where((ids >= 0) & (ids < rows), ids, rows)
    order = np.argsort(key, kind="stable")
    order = order[: int((key < rows).sum())]
    longest = np.flatnonzero(key[order] == np.bincount(key[order]).argmax())
    eighth = (longest.size + 7) // 8
    chunk = 16 if n <= 1 << 17 else 64 if n <= 1 << 20 else 256
    chunks = (order.size + chunk - 1) // chunk
    for lost in (order[:chunk], order[chunks // 2 * chunk:][:chunk], order[(chunks - 1) * chunk:], order[longest[3 * eighth: 4 * eighth]],
                 order[longest[:1]]):
        missing = np.stack([np.bincount(ids[lost], weights=column[lost], minlength=rows) for column in grad.T], 1)
        assert np.all((missing > 0).any(0))
        assert not np.array_equal(sums - missing, sums)
