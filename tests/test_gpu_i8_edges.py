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


@pytest.mark.parametrize("E", [128, 1024])
@pytest.mark.parametrize("bf16", [False, True])
def test_softmax_weights_of_many_equal_logits(E, bf16):
    """one expert ahead and the rest at one logit: the errors of the exponentials are the same and add up. The weights that are not renormalised carry the sum's error, 4e-7 at
    most, and one rounding of their own"""
    import torch
    g = torch.Generator(device="cuda"); g.manual_seed(E)
    T = 40000
    top = torch.rand(T, generator=g, device="cuda") * 4 - 2
    l = (top - 3 - 5 * torch.rand(T, generator=g, device="cuda"))[:, None].repeat(1, E)
    l[torch.arange(T, device="cuda"), torch.randint(E, (T,), generator=g, device="cuda")] = top
    if bf16:
        l = l.bfloat16()
    for K in (1, 3):
        ids, w = torch.zeros((T, K), dtype=torch.int32, device="cuda"), torch.zeros((T, K), device="cuda")
        ok(api.lib.omega_gpu_moe_route_async(api.MoeRouteConfig(E, K, api.SCORE_SOFTMAX, 1, 0, 1, 0, 1.0), T, l.data_ptr(), int(bf16), 0, 0, ids.data_ptr(), w.data_ptr(), here()))
        want = torch.softmax(l.double(), 1).gather(1, ids.long())
        assert torch.equal(ids[:, 0].long(), l.argmax(1))
        assert float(((w.double() - want).abs() / want).max()) <= 4e-7 + EPS24


def test_softmax_of_logits_whose_difference_is_no_number():
    """the largest and the lowest value of the type, infinities: no NaN from the difference's own rounding"""
    big = np.finfo(np.float32).max
    l = np.full((4, 64), -3.0, np.float32)
    l[0] = -big; l[0, 7] = big; l[1, 9] = np.inf; l[2, ::2] = -np.inf; l[2, 3] = big; l[3] = -big; l[3, 5] = 2e38
    for norm in (0, 1):
        rc, ids, w = api.moe_route(api.MoeRouteConfig(64, 3, api.SCORE_SOFTMAX, 1, 0, 1, norm, 1.0), l); ok(rc)
        want, wants = ref.route(l, 3, False, norm=bool(norm))
        assert np.array_equal(ids, want) and np.array_equal(w, wants)


@pytest.mark.parametrize("E", [128, 1024])
def test_softmax_picks_next_to_a_tie_of_score_and_bias(E):
    """one expert ahead, the rest at one logit, and a bias that lifts another expert to where the two change places as the logit ahead goes through neighbouring floats"""
    for base, low in ((0.95, -4.92), (0.0, -5.9), (-1.5, -6.5)):
        l = np.full((240, E), low, np.float32)
        l[:, 9] = (np.float32(base).view(np.uint32) + np.arange(240, dtype=np.uint32) * 2).view(np.float32) if base else np.linspace(-1e-5, 1e-5, 240).astype(np.float32)
        p = np.exp(l[120].astype(np.float64)); p /= p.sum()
        bias = np.zeros(E, np.float32); bias[4] = p[9] - p[4]
        rc, ids, w = api.moe_route(api.MoeRouteConfig(E, 2, api.SCORE_SOFTMAX, 1, 0, 1, 1, 1.0), l, bias); ok(rc)
        want, _ = ref.route(l, 2, False, bias)
        assert np.array_equal(ids, want) and len(set(ids[:, 0].tolist())) == 2


# ------------------------------------------------------------------ the layer
@pytest.mark.parametrize("T,E,H,I,K", [(1, 1, 16, 16, 1), (3, 1, 16, 16, 1), (70, 2, 16, 48, 2), (1, 1024, 64, 32, 32), (40, 1024, 64, 32, 32), (300, 1024, 64, 32, 16), (1, 40, 16, 8192, 32), (2, 2, 16384, 16, 1)])
def test_layer_of_extreme_shapes(T, E, H, I, K):
    from tests.test_gpu_i8 import Layer, bits, check_rows, quantised
    L = Layer(T + E, E, H, I, K, T)
    rng = np.random.default_rng(T)
    lg, x = bits(rng.normal(0, 1, (T, E)).astype(np.float32)), bits(rng.normal(0, 1, (T, H)).astype(np.float32))
    rc, o16, o32, ids, w = api.moe_i8_layer_bf16(L.h, lg, x, K); ok(rc)
    q, s = quantised(x)
    check_rows(q, s, api.bf16_to_f32(x).astype(np.float64), 0.0)
    wids, ww, want = L.want(lg, q, s)
    assert np.array_equal(ids, wids) and np.all(np.abs(w - ww) <= (K + 5) * EPS24 * ww)
    # A code may fall one step off with a chance of 127 * 2 * 2e-6 + 1.3e-4 (see LAYER_REL); as many of the I T K codes as that makes likely, and four deviations and one more. The codes' rms is
    # 30 or more in short rows; in one of thousands the largest of the products is further out, 8
    n = I * T * K; mean = n * (127 * 2 * 2e-6 + 1.3e-4)
    off = np.ceil(mean + 4 * np.sqrt(mean) + 1)
    assert np.linalg.norm(o32 - want) <= np.sqrt(off / n) / (30 if I <= 256 else 8) * np.linalg.norm(want)
    L.free()


def test_layer_rows_that_are_not_finite_stay_by_themselves():
    from tests.test_gpu_i8 import Layer, bits
    for T, E, K in ((40, 8, 2), (700, 8, 8)):
        L = Layer(3, E, 256, 128, K, T)
        rng = np.random.default_rng(T)
        lg, x = bits(rng.normal(0, 1, (T, E)).astype(np.float32)), bits(rng.normal(0, 1, (T, 256)).astype(np.float32))
        rc, _, want, _, _ = api.moe_i8_layer_bf16(L.h, lg, x, K); ok(rc)
        want = want.copy()
        bad = x.copy(); bad[5, 17] = 0x7fc0; bad[11, 3] = 0x7f80; bad[T - 1, 0] = 0xff80
        rc, o16, o32, _, _ = api.moe_i8_layer_bf16(L.h, lg, bad, K); ok(rc)
        rest = np.ones(T, bool); rest[[5, 11, T - 1]] = False
        assert np.isnan(o32[~rest]).all() and np.isnan(api.bf16_to_f32(o16[~rest])).all()
        assert np.array_equal(o32[rest].view(np.uint32), want[rest].view(np.uint32))
        L.free()


def test_captured_layer_between_eager_calls_of_other_sizes():
    """a step of 700 tokens and one of one token, captured; between their replays the same layer runs 1024, 600 and 3 tokens"""
    import torch
    from tests.test_gpu_i8 import Layer
    E, H, I, K, most = 8, 256, 128, 8, 1024
    L = Layer(7, E, H, I, K, most)
    g = torch.Generator(device="cuda"); g.manual_seed(2)
    lg, x = torch.randn((most, E), generator=g, device="cuda").bfloat16(), torch.randn((most, H), generator=g, device="cuda").bfloat16()
    out = {n: torch.zeros((n, H), device="cuda") for n in (700, 1, 1024, 600, 3)}

    def call(n):
        ok(api.lib.omega_gpu_moe_i8_layer_async(L.h, n, lg.data_ptr(), x.data_ptr(), out[n].data_ptr(), 0, here()))
    want = {}
    for n in out:
        call(n); torch.cuda.synchronize(); want[n] = out[n].clone()
    graphs = {}
    for n in (700, 1):
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n]):
            call(n)
    for n in (700, 1024, 700, 1, 600, 700, 700, 3, 1, 1024, 600, 700):
        out[n].fill_(-7)
        graphs[n].replay() if n in graphs else call(n)
        torch.cuda.synchronize()
        assert torch.equal(out[n], want[n]) and api.lib.omega_gpu_moe_i8_layer_status(L.h, here()) == 0
    L.free()


def test_two_layers_on_the_same_tensors_at_once():
    import torch
    from tests.test_gpu_i8 import Layer, config
    E, H, I, K = 16, 512, 256, 4
    L = Layer(9, E, H, I, K, 400)
    rc, other = api.moe_i8_layer_create(L.tgu, L.tdn, config(E, K, True), L.bias, 30); ok(rc)
    g = torch.Generator(device="cuda"); g.manual_seed(4)
    jobs = []
    for h, T in ((L.h, 400), (other, 30)):
        lg, x = torch.randn((T, E), generator=g, device="cuda").bfloat16(), torch.randn((T, H), generator=g, device="cuda").bfloat16()
        jobs.append((h, T, lg, x, [torch.zeros((T, H), device="cuda") for _ in range(30)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(30):
        for h, T, lg, x, outs, s in jobs:
            ok(api.lib.omega_gpu_moe_i8_layer_async(h, T, lg.data_ptr(), x.data_ptr(), outs[i].data_ptr(), 0, s.cuda_stream))
    torch.cuda.synchronize()
    for h, T, lg, x, outs, s in jobs:
        assert outs[0].any() and all(torch.equal(outs[0], o) for o in outs[1:]) and api.lib.omega_gpu_moe_i8_layer_status(h, here()) == 0
    api.lib.omega_gpu_moe_i8_layer_free(other)
    L.free()
