"""The 8-bit integer path at calls that a plan, a size or a value makes unusual."""
import numpy as np
import pytest

from cudapp_b200 import api
from tests import i8_reference as ref
from tests.i8_reference import EPS24
from tests.test_gpu_i8 import codes, dev, here, ok, scales

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile_rows", [5, 40, 160])
@pytest.mark.parametrize("gathered", [True, False])
@pytest.mark.parametrize("n", [264, 100])
def test_grouped_product_of_a_plan_that_does_not_fit(tile_rows, gathered, n):
    """tiles with more rows than tile_rows, and rows past x_rows: the tile is cut there, and nothing else is written. The buffers hold all of the plan's rows"""
    import torch
    rng = np.random.default_rng(tile_rows + n)
    E, k, R, x_rows = 3, 256, 512, 300
    first, rows, experts = [0, 175, 280, 296, 299, 310], [tile_rows + 9, min(tile_rows, 100), 15, 3, 7, 20], [1, 0, 2, 7, 1, 0]   # expert 7: the last one
    tiles = np.zeros((len(rows), 4), np.uint32)
    tiles[:, 0], tiles[:, 1], tiles[:, 2] = experts, first, rows
    x, xs, w, ws = codes(rng, R, k), scales(rng, R), codes(rng, E * n, k), scales(rng, E * n)
    xmap, ymap = rng.integers(0, 2 * x_rows, R).astype(np.uint32), rng.permutation(R).astype(np.uint32)
    rc, t = api.i8_upload(w, ws); ok(rc)
    y, y16 = torch.full((R, n), 3.0, device="cuda"), torch.full((R, n), 3.0, dtype=torch.bfloat16, device="cuda")
    dt, dh, dx, dxs, dxm, dym = dev(tiles), dev(np.array([0, 0, len(rows), 0], np.uint32)), dev(x), dev(xs), dev(xmap), dev(ymap)
    for a, b in ((y.data_ptr(), 0), (0, y16.data_ptr())):
        ok(api.lib.omega_gpu_i8_gemm_grouped_async(t, E, tile_rows, len(rows), dt.data_ptr(), dh.data_ptr(), dxm.data_ptr() if gathered else 0, dym.data_ptr(), dx.data_ptr(), x_rows,
                                                   dxs.data_ptr(), b, a, here()))
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    want = np.full((R, n), 3.0)
    for e, r0, c in zip(experts, first, rows):
        e = min(e, E - 1)
        for r in range(r0, r0 + min(c, tile_rows)):
            if gathered or r < x_rows:
                src = min(xmap[r], x_rows - 1) if gathered else r
                want[ymap[r]] = ref.gemm(x[src:src + 1], xs[src:src + 1], w[e * n:(e + 1) * n], ws[e * n:(e + 1) * n])[0]
    assert np.all(np.abs(y.cpu().numpy() - want) <= 3 * EPS24 * np.abs(want))
    assert np.all(np.abs(y16.double().cpu().numpy() - want) <= (2.0 ** -8 * (1 + 2 ** -7) + 4 * EPS24) * np.abs(want))
    api.lib.omega_gpu_i8_free(t)
