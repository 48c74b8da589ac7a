"""The cases of rows that end inside a vector can fail: sums in which the shared columns count twice, or are missing, lie far
outside of what the GPU tests allow.  The mistake is planted in the 64-bit forms; no GPU is touched."""

import pytest
import torch

import int8_ref as R


@pytest.mark.parametrize("dtype", R.DTYPES, ids=R.IDS)
@pytest.mark.parametrize("cols", R.RAGGED)
def test_a_column_counted_twice_or_not_at_all_is_seen(cols, dtype):
    shared = list(range(cols - 8, cols - cols % 8))
    for at in R.loud_places(cols):
        if at not in shared:
            continue
        h, g, w = R.loud_row(cols, at, dtype, dtype)
        _, r, rel_r, _ = R.norm(h, w, 1e-6)
        rstd = r.float()
        want, allowed, _, _ = R.norm_backward(g, h, rstd, w, None, dtype, dtype)
        for times in (2.0, 0.0):
            count = torch.ones(cols, dtype=torch.float64)
            count[shared] = times
            hd, gd, wd, rd = h.double(), g.double(), w.double(), rstd.double()[:, None]
            wrong_r = 1 / torch.sqrt((hd.square() * count).sum(1) / cols + 1e-6)
            assert bool(((wrong_r - r).abs() > 10 * rel_r * r).all())
            gw, xhat = gd * wd, hd * rd
            wrong = rd * (gw - xhat * (gw * xhat * count).mean(1, keepdim=True))
            assert bool(((wrong - want).abs() > 10 * allowed)[:, at].all())
