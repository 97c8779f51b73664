"""How far the training-side operators' sums may be off by their real depth: long sums of terms of one sign, whose roundings add
up where they are all made in one 32-bit accumulator."""
import numpy as np
import pytest

import training_reference as ref
from test_gpu_backward_rows import KINDS, run_layernorm_backward

pytestmark = pytest.mark.gpu

U = ref.U


# (rows, columns): through the column kernel alone where there is no workspace, where rows are shorter than a vector and where they
# are longer than the registers; else through the row kernel
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(786432, 24), (200000, 40), (300001, 3), (70000, 130), (6000, 17000)])
def test_column_sums_over_many_rows(ko, rows, cols, kind):
    rng = np.random.default_rng(rows + cols)
    dy, dy64 = ref.to_storage(rng.uniform(0.5, 1.0, (rows, cols)).astype(np.float32), kind)
    x, x64 = ref.to_storage(rng.uniform(1.0, 2.0, (rows, cols)).astype(np.float32), kind)
    mean, rstd = np.full(rows, 0.25, np.float32), np.full(rows, 1.5, np.float32)
    want_g, want_b = (dy64 * ((x64 - 0.25) * 1.5)).sum(0), dy64.sum(0)
    for workspace in (True, False):
        _, dgamma, dbeta = run_layernorm_backward(ko, dy, x, mean, rstd, kind, workspace=workspace)
        # without a workspace: eight terms in 32 bits, then 64, and one rounding.  With one: eight terms likewise, or a lane group's
        # rows one after the other (512 workgroups of 4 wavefronts with 8 lane groups of 8 lanes: rows / 16384; rows of 130 columns
        # 16 to 64 lanes, rows / 2048 at least), 32 lane groups, and the partial rows, eight of them in turn and a tree of 64 lanes
        depth = 8 + 1 if not workspace else max(8, rows / (16384 if cols <= 64 else 2048)) + 32 + 8 + 6
        # xh carries two roundings, its product with dy one
        ref.assert_within(dgamma, want_g, (depth + 3) * U * want_g, "dgamma, workspace %s" % workspace)
        ref.assert_within(dbeta, want_b, depth * U * want_b, "dbeta, workspace %s" % workspace)
