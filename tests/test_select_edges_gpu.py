"""Edges of the choice of blocks by score."""
from __future__ import annotations

import pytest
import torch

import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("nbk", [8, 200, 700])
@pytest.mark.parametrize("cu", [[2 ** 31 - 1, -2 ** 31, -2 ** 31 + 1], [5, 4, 5], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]])
def test_row_ranges_that_make_no_sense_keep_nothing(nbk, cu):
    """Also where their difference wraps to one new token, as a sequence might have."""
    scores = torch.rand(2, 4, 2, nbk, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = T.select_blocks(scores, 2, torch.tensor(cu, device=DEV).to(torch.int32),
                           torch.tensor([300, 400], dtype=torch.int32, device=DEV), 3, err=err)
    assert int(err.item()) == 1
    assert (kept.cnt[0] == 0).all() and (kept.idx[0] == -1).all()
