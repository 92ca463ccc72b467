"""Edges of the batched serving operators: contents, lengths, aliases and plans that the parity tests do not reach."""

import numpy as np
import pytest
import torch

import batch_ref as R
from test_batch_gpu import DEV, _attend_case, _dev, _f64, _run_attend, q4b  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- prefix_attention: what stands behind the last key ------------------------------------------------


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,g,page", [(1, 3, 16), (1, 8, 64), (3, 5, 8), (2, 8, 24), (20, 4, 16), (30, 8, 64)])
def test_rest_of_a_page_never_shows(q4b, hd, new, g, page):  # noqa: F811
    """Own keys that end at every place of a 64-key (and of a 128-key) tile, NaN keys and infinite values behind them, in
    the narrow kernel (few rows a sequence) and the tensor-core one (more than 64 rows x heads), again and again over the
    same shared memory."""
    lens = [(new, max(n, new)) for n in range(1, 131)]
    case = _attend_case(lens, page, 0, 2 * g, 2, hd, torch.float16, seed=page + g)
    out, _, live = _run_attend(q4b, case, page)
    assert live.all() and bool(torch.isfinite(out).all())
