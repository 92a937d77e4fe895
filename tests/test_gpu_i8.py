"""The 8-bit integer path on the GPU against its definitions in 64 bits: routing by scores, residual + RMSNorm and SiLU gate to 8-bit rows, the product (plain and
grouped by expert), the layer, and a run of them together. Tolerances count roundings to f32 (2^-24 each, relative) and, where a result is bf16, its one of 2^-8."""
import ctypes as C

import numpy as np
import pytest

from cudapp_b200 import api
from tests import i8_reference as ref
from tests.i8_reference import EPS24

pytestmark = pytest.mark.gpu
BF16_HALF = 2.0 ** -8


def ok(rc):
    assert rc == 0, api.last_error()


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    view = {np.dtype(np.uint32): np.int32, np.dtype(np.uint16): np.int16}.get(a.dtype)
    return torch.from_numpy(a.view(view) if view else a).to("cuda:0")


def here():
    import torch
    return torch.cuda.current_stream().cuda_stream


def bits(x):
    return api.bf16_bits(x)


# ------------------------------------------------------------------ routing
def config(E, topk, sigmoid, groups=1, kept=0, rank=1, norm=True, scale=1.0):
    return api.MoeRouteConfig(E, topk, api.SCORE_SIGMOID if sigmoid else api.SCORE_SOFTMAX, groups, kept, rank, int(norm), scale)


def check_route(logits, bias, E, topk, sigmoid, groups=1, kept=0, rank=1, norm=True, scale=1.0, bf16=False):
    stored = bits(logits) if bf16 else np.asarray(logits, np.float32)
    rc, ids, w = api.moe_route(config(E, topk, sigmoid, groups, kept, rank, norm, scale), stored, bias); ok(rc)
    want, wants = ref.route(api.bf16_to_f32(stored) if bf16 else stored, topk, sigmoid, bias, groups, kept, rank, norm, scale)
    assert np.array_equal(ids, want)
    # scores rounded once, a sum of topk of them, a quotient, a product
    assert np.all(np.abs(w - wants) <= (topk + 5) * EPS24 * np.abs(wants) + 1e-44)
    return ids, w


@pytest.mark.parametrize("E,topk,groups,kept,rank", [(1, 1, 1, 0, 1), (8, 2, 1, 0, 1), (60, 4, 4, 2, 2), (64, 6, 8, 3, 2), (100, 8, 4, 1, 1), (128, 8, 1, 0, 1), (128, 8, 32, 5, 2), (160, 6, 8, 3, 1),
                                                      (256, 8, 8, 4, 2), (256, 32, 8, 2, 2), (257, 5, 1, 0, 1), (384, 8, 8, 8, 2), (512, 8, 16, 4, 2), (1000, 10, 20, 3, 2), (1024, 32, 32, 1, 2)])
@pytest.mark.parametrize("sigmoid,biased,bf16", [(True, True, False), (True, False, True), (False, False, False), (False, True, True)])
def test_route(E, topk, groups, kept, rank, sigmoid, biased, bf16):
    rng = np.random.default_rng(E * 8 + topk + sigmoid)
    bias = rng.normal(0, 0.1, E).astype(np.float32) if biased else None
    for T in (1, 5, 67):
        check_route(rng.normal(0, 1.5, (T, E)).astype(np.float32), bias, E, topk, sigmoid, groups, kept, rank, norm=T != 5, scale=2.5 if T == 5 else 1.0, bf16=bf16)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("E,groups,kept", [(64, 1, 0), (64, 8, 2), (60, 4, 2)])
def test_route_ties_masks_and_values_that_are_no_numbers(sigmoid, E, groups, kept):
    rng = np.random.default_rng(E + groups)
    l = np.round(rng.normal(0, 1, (24, E)), 0).astype(np.float32)          # many ties
    l[0] = 0.0                                                              # one score for all
    l[1] = -np.inf                                                          # a mask that leaves nothing
    l[2] = np.nan
    l[3, ::2] = -np.inf                                                     # half masked
    l[4, ::3] = np.nan
    l[5, 7] = np.inf
    l[6, [3, 9, 40]] = np.inf
    l[7] = np.finfo(np.float32).min                                         # masked by the type's lowest value
    l[8, 5:] = np.finfo(np.float32).min
    l[9] = -np.inf; l[9, 11] = np.nan; l[9, 12] = -3.0
    l[10] = 1e30; l[11] = -1e30
    bias = np.zeros(E, np.float32); bias[4] = -np.inf; bias[20] = 0.5
    for b in (None, bias):
        for norm in (True, False):
            ids, w = check_route(l, b, E, 6, sigmoid, groups, kept, 2 if groups > 1 else 1, norm=norm)
            assert all(len(set(r)) == 6 for r in ids.tolist()) and np.isfinite(w).all()
            assert not w[1].any() and not w[2].any()


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("E,groups,kept", [(256, 8, 4), (128, 1, 0), (60, 4, 2), (600, 1, 0)])
def test_route_scores_a_unit_in_the_last_place_apart(sigmoid, biased, E, groups, kept):
    """logits that are neighbours among the floats, that saturate the sigmoid, or whose softmax is subnormal: f32 scores cannot order them, 64 bits can"""
    rng = np.random.default_rng(E + sigmoid)
    l = np.empty((10, E), np.float32)
    for t, (base, step) in enumerate([(0.7, 1), (0.7, 3), (2.5, 1), (-3.0, 2), (16.9, 40), (30.0, 1), (-20.0, 1)]):
        l[t] = (np.float32(base).view(np.uint32) + rng.permutation(E).astype(np.uint32) * step).view(np.float32)
    l[7] = rng.normal(-60, 8, E); l[7, 5] = 40.0                             # one expert takes it all
    l[8] = np.repeat(rng.normal(0, 1, E // 4), 4)[:E]                        # ties in fours
    l[9] = rng.normal(0, 1e-6, E)
    bias = (rng.integers(-3, 3, E) * 0.25).astype(np.float32) if biased else None
    for topk in (1, 6, 32):
        if topk <= (kept or groups) * (E // groups):
            check_route(l, bias, E, topk, sigmoid, groups, kept, 2 if groups > 1 else 1)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("E,groups,kept", [(24, 1, 0), (64, 1, 0), (256, 8, 4), (600, 1, 0)])
def test_route_picks_among_scores_below_the_normal_numbers(sigmoid, E, groups, kept):
    """no bias, and picks whose scores are a few units of the smallest float: many are equal once rounded, and the lowest index has to come first"""
    rng = np.random.default_rng(E)
    l = np.empty((60, E), np.float32)
    for t in range(60):
        l[t] = rng.uniform(-103.5, -86.0, E) if t % 2 else -95.0 + rng.uniform(0, 2e-3, E)
        if not sigmoid:
            l[t] += 90.0
            l[t, :: max(1, E // 3)] = 90.0                                   # three or four take it all
    for topk in (2, 8, 20):
        if topk <= (kept or groups) * (E // groups):
            check_route(l, None, E, topk, sigmoid, groups, kept, 2 if groups > 1 else 1)


def test_route_softmax_scores_that_round_to_the_same_tiny_float():
    """seven clear picks, and an eighth among two dozen scores of 48 to 51 units of the smallest float: equal once rounded, though a rounded exponential times a rounded factor is not"""
    rng = np.random.default_rng(8)
    l = np.full((400, 128), -np.inf, np.float32)
    for t in range(400):
        at = rng.permutation(np.arange(0, 128, 4))
        l[t, at[:7]] = (90.0, 89.9, 89.7, 60.0, 50.0, 40.0, 30.0)
        total = np.exp(l[t, at[:7]].astype(np.float64) - 90.0).sum()
        l[t, at[7:]] = 90.0 + np.log(total * rng.uniform(48.3, 50.7, 25) * 2.0 ** -149)
    check_route(l, None, 128, 8, False)


def test_route_strided_rows_on_another_stream():
    import torch
    rng = np.random.default_rng(5)
    T, E, pad = 33, 96, 13
    for bf16 in (False, True):
        wide = rng.normal(0, 1, (T, E + pad)).astype(np.float32)
        stored = bits(wide) if bf16 else wide
        want, _ = ref.route((api.bf16_to_f32(stored) if bf16 else stored)[:, 3:3 + E], 6, True, None, 8, 4, 2)
        s, d = torch.cuda.Stream(), dev(stored)
        ids, w = torch.full((T + 1, 6), -7, dtype=torch.int32, device="cuda"), torch.zeros((T, 6), device="cuda")
        torch.cuda.synchronize()
        size = 2 if bf16 else 4
        ok(api.lib.omega_gpu_moe_route_async(config(E, 6, True, 8, 4, 2), T, d.data_ptr() + 3 * size, int(bf16), (E + pad) * size, 0, ids.data_ptr(), w.data_ptr(), s.cuda_stream))
        s.synchronize()
        assert np.array_equal(ids[:T].cpu().numpy().view(np.uint32), want) and (ids[T] == -7).all()


# ------------------------------------------------------------------ 8-bit rows
def check_rows(q, s, y, rel):
    """codes and scales against unrounded float64 rows whose f32 counterparts are off by at most `rel`: the largest value and the quotient each carry it"""
    v, want = ref.quant(y)
    assert np.array_equal(np.isnan(s), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.all(np.abs(s[fine] - want[fine]) <= (rel + EPS24) * want[fine])
    assert np.all(np.abs(q - v) <= 0.5 + 127 * (2 * rel + 4 * EPS24)) and np.abs(q.astype(np.int32)).max() <= 127
    assert not q[~fine].any()


@pytest.mark.parametrize("T,H", [(1, 16), (3, 48), (5, 512), (4, 528), (2, 2048), (7, 2064), (2, 4096), (3, 5008), (2, 8192), (1, 16384), (600, 256)])
@pytest.mark.parametrize("x16,m,weighted", [(False, "f32", True), (True, None, False), (True, "bf16", True), (False, "bf16", False), (False, None, True), (True, "f32", True)])
def test_norm(T, H, x16, m, weighted):
    import torch
    rng = np.random.default_rng(T * H)
    x = rng.normal(0, 2, (T, H)).astype(np.float32); d = rng.normal(0, 1, (T, H)).astype(np.float32); w = rng.normal(1, 0.3, H).astype(np.float32)
    dx, dm, dw = dev(bits(x) if x16 else x), None if m is None else dev(bits(d) if m == "bf16" else d), dev(w)
    h = ref.bf16(x) if x16 else x.astype(np.float64)
    if m:
        h = h + (ref.bf16(d) if m == "bf16" else d)
    h = h.astype(np.float32).astype(np.float64)                             # the residual is f32: one rounding, the same here and there
    out, q, s = torch.zeros((T, H), device="cuda"), torch.full((T + 1, H), 55, dtype=torch.int8, device="cuda"), torch.zeros(T, device="cuda")
    xn = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, dx.data_ptr() if x16 else 0, dm.data_ptr() if m else 0, int(m == "bf16"), 0 if x16 else dx.data_ptr(), out.data_ptr(),
                                                dw.data_ptr() if weighted else 0, xn.data_ptr(), q.data_ptr(), s.data_ptr(), here()))
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy().astype(np.float64), h) and (q[T] == 55).all()
    y = ref.norm(h, w if weighted else None, 1e-6)
    check_rows(q[:T].cpu().numpy(), s.cpu().numpy(), y, 4 * EPS24)          # the factor, two products, one for the largest value
    assert np.all(np.abs(xn.double().cpu().numpy() - y) <= (BF16_HALF + 4 * EPS24) * np.abs(y))
    # in place, without the optional outputs: the same codes
    if not x16:
        q2 = torch.zeros_like(q)
        ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, 0, dm.data_ptr() if m else 0, int(m == "bf16"), dx.data_ptr(), dx.data_ptr(), dw.data_ptr() if weighted else 0, 0, q2.data_ptr(),
                                                    s.data_ptr(), here()))
        assert torch.equal(q2[:T], q[:T]) and torch.equal(dx, out)
        ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, 0, 0, 0, out.data_ptr(), 0, dw.data_ptr() if weighted else 0, 0, q2.data_ptr(), s.data_ptr(), here()))
        assert torch.equal(q2[:T], q[:T])


@pytest.mark.parametrize("H", [48, 2048])
def test_norm_rows_at_the_edges(H):
    rng = np.random.default_rng(H)
    x = rng.normal(0, 1, (9, H)).astype(np.float32)
    x[0] = 0.0; x[1, 5] = np.nan; x[2, 7] = np.inf; x[3, H - 1] = -np.inf
    x[4] *= np.float32(1e25); x[5] *= np.float32(1e-30); x[6, :] = 0; x[6, 3] = 4.0; x[7] = np.float32(3e38)
    w = np.ones(H, np.float32); w[7] = 0                                     # 0 * infinity
    rc, h, q, s = api.residual_norm_q8_f32(x, None, w); ok(rc)
    assert np.array_equal(h.view(np.uint32), x.view(np.uint32))
    y = ref.norm(x.astype(np.float64), w, 1e-6)
    y[[1, 2, 3]] = np.nan
    check_rows(q, s, y, 4 * EPS24)
    assert s[0] == np.float32(2.0 ** -100 / 127) and np.isnan(s[[1, 2, 3]]).all() and np.isfinite(s[[4, 7]]).all()
    rc, _, _, s0 = api.residual_norm_q8_f32(x[:1], None, None, eps=0.0); ok(rc)
    assert np.isnan(s0[0])                                                   # 0 / 0


@pytest.mark.parametrize("H", [16, 2048])
def test_norm_of_tiny_rows_without_eps(H):
    """mean squares whose root's reciprocal leaves the f32 range"""
    rng = np.random.default_rng(H)
    x = rng.normal(0, 1, (5, H)).astype(np.float32) * np.float32([1e-20, 1e-30, 1e-37, 1e-39, 1e-42])[:, None]
    rc, _, q, s = api.residual_norm_q8_f32(x, None, None, eps=0.0); ok(rc)
    check_rows(q, s, ref.norm(x.astype(np.float64), None, 0.0), 4 * EPS24)


# the fast exponential is off by (2 + 1.173 |g|) 2^-23, its quotient by 2 more units, the product by one rounding
GATE_REL = lambda g: ((2 + 1.173 * g) + 2) * 2.0 ** -23 + EPS24              # noqa: E731


@pytest.mark.parametrize("rows,inter", [(1, 16), (9, 48), (3, 256), (17, 272), (8, 512), (5, 768), (1000, 768), (3, 1024), (2, 1040), (3, 2064), (2, 5008), (1, 16384)])
@pytest.mark.parametrize("bf16", [True, False])
def test_gate(rows, inter, bf16):
    import torch
    rng = np.random.default_rng(rows + inter)
    gu = np.clip(rng.normal(0, 2, (rows, 2 * inter)), -8, 8).astype(np.float32)
    d = dev(bits(gu) if bf16 else gu)
    y = ref.gate(ref.bf16(gu) if bf16 else gu)
    q, s = torch.full((rows + 1, inter), 55, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    ok(api.lib.omega_gpu_swiglu_q8_async(rows, inter, d.data_ptr(), int(bf16), q.data_ptr(), s.data_ptr(), here()))
    check_rows(q[:rows].cpu().numpy(), s.cpu().numpy(), y, GATE_REL(8)); assert (q[rows] == 55).all()
    # the same rows without the gate, a stride apart
    wide = dev(bits(gu) if bf16 else gu)
    ok(api.lib.omega_gpu_quant_q8_async(rows, inter, wide.data_ptr() + inter * (2 if bf16 else 4), int(bf16), 2 * inter * (2 if bf16 else 4), q.data_ptr(), s.data_ptr(), here()))
    check_rows(q[:rows].cpu().numpy(), s.cpu().numpy(), (ref.bf16(gu) if bf16 else gu.astype(np.float64))[:, inter:], 0.0)


def test_gate_rows_at_the_edges():
    rng = np.random.default_rng(3)
    I = 128
    gu = rng.normal(0, 1, (8, 2 * I)).astype(np.float32)
    gu[0] = 0; gu[1, 4] = np.nan; gu[2, I + 9] = np.inf; gu[3, 7] = -np.inf; gu[4, :I] = -200.0; gu[5, :I] = 100.0; gu[6, 3] = np.inf
    rc, q, s = api.swiglu_q8_f32(gu); ok(rc)
    y = ref.gate(gu); y[[1, 2, 3, 6]] = np.nan; y[4] = 0                      # -200: a gate of 1e-87 is below the least row
    check_rows(q, s, y, GATE_REL(100))
    assert np.isnan(s[[1, 2, 3, 6]]).all() and not q[4].any()


# ------------------------------------------------------------------ the product
def codes(rng, *shape):
    return rng.integers(-127, 128, shape).astype(np.int8)


def scales(rng, n, about=0.01):
    return (rng.uniform(0.5, 1.5, n) * about).astype(np.float32)


def check_product(y16, y32, want):
    bound = 3 * EPS24 * np.abs(want)                                          # the sum, the product of the scales, the product
    assert np.all(np.abs(y32 - want) <= bound)
    assert np.all(np.abs(api.bf16_to_f32(y16) - want) <= BF16_HALF * np.abs(want) * (1 + 2 ** -7) + bound)


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 130, 257, 520])
@pytest.mark.parametrize("n,k", [(1, 16), (16, 64), (17, 48), (100, 112), (128, 128), (129, 144), (256, 2048), (1000, 528), (300, 4112)])
def test_product(m, n, k):
    rng = np.random.default_rng(m * n + k)
    x, xs, w, ws = codes(rng, m, k), scales(rng, m), codes(rng, n, k), scales(rng, n)
    rc, t = api.i8_upload(w, ws); ok(rc)
    rc, y16, y32 = api.i8_gemm(t, n, x, xs); ok(rc)
    check_product(y16, y32, ref.gemm(x, xs, w, ws))
    api.lib.omega_gpu_i8_free(t)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_of_extreme_codes_and_rows_that_are_not_finite(m):
    n, k = 48, 32768
    rng = np.random.default_rng(m)
    x, w = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    w[1::2] = 127
    xs, ws = np.ones(m, np.float32), np.ones(n, np.float32)
    xs[-1] = np.nan
    x[0, :17] = rng.integers(-128, 128, 17)
    rc, t = api.i8_upload(w, ws); ok(rc)
    rc, y16, y32 = api.i8_gemm(t, n, x, xs); ok(rc)
    want = ref.gemm(x, xs, w, ws)
    assert np.isnan(y32[-1]).all() and np.isnan(api.bf16_to_f32(y16[-1])).all()
    if m > 1:
        check_product(y16[:-1], y32[:-1], want[:-1])
        assert y32[1, 0] == 2.0 ** 29
    api.lib.omega_gpu_i8_free(t)


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (20, 100, 512), (200, 384, 1040)])
def test_product_on_device_rows_a_stride_apart(m, n, k):
    """weights from the device, rows inside wider ones, one output only, another stream, what lies behind the last row left alone"""
    import torch
    rng = np.random.default_rng(k)
    wide, xs, w, ws = codes(rng, m, k + 32), scales(rng, m), codes(rng, n, k), scales(rng, n)
    dw, dws, dx, dxs = dev(w), dev(ws), dev(wide), dev(xs)
    rc, t = api.i8_upload_dev(n, k, dw.data_ptr(), dws.data_ptr()); ok(rc)
    dw.zero_(); dws.zero_()                                                   # copied
    s = torch.cuda.Stream()
    y16, y32 = torch.full((m + 1, n), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((m + 1, n), 3.0, device="cuda")
    torch.cuda.synchronize()
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, dx.data_ptr() + 16, k + 32, dxs.data_ptr(), y16.data_ptr(), 0, s.cuda_stream))
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, dx.data_ptr() + 16, k + 32, dxs.data_ptr(), 0, y32.data_ptr(), s.cuda_stream))
    s.synchronize()
    check_product(y16[:m].cpu().view(torch.int16).numpy().view(np.uint16), y32[:m].cpu().numpy(), ref.gemm(wide[:, 16:16 + k], xs, w, ws))
    assert (y16[m] == 3).all() and (y32[m] == 3).all()
    api.lib.omega_gpu_i8_free(t)


@pytest.mark.parametrize("m,n,k", [(1100, 4104, 4112), (4136, 2056, 2064), (2049, 4096, 1024), (900, 4090, 3600)])
def test_large_products(m, n, k):
    """pairs of CTAs and their ragged ends; the reference in 64 bits on the GPU"""
    import torch
    g = torch.Generator(device="cuda"); g.manual_seed(m)
    x, w = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8, device="cuda") for s in ((m, k), (n, k)))
    xs, ws = torch.rand(m, generator=g, device="cuda") + 0.5, torch.rand(n, generator=g, device="cuda") + 0.5
    rc, t = api.i8_upload_dev(n, k, w.data_ptr(), ws.data_ptr()); ok(rc)
    y16, y32 = torch.full((m + 1, n), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((m + 1, n), 3.0, device="cuda")
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, x.data_ptr(), 0, xs.data_ptr(), y16.data_ptr(), 0, here()))
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, x.data_ptr(), 0, xs.data_ptr(), 0, y32.data_ptr(), here()))
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    want = (x.double() @ w.double().T) * torch.outer(xs.double(), ws.double())
    assert bool(((y32[:m].double() - want).abs() <= 3 * EPS24 * want.abs()).all()) and torch.equal(y16[:m], y32[:m].bfloat16())
    assert bool((y16[m] == 3).all()) and bool((y32[m] == 3).all())
    api.lib.omega_gpu_i8_free(t)


@pytest.mark.parametrize("m,n,k", [(300, 1024, 1936), (130, 6144, 1008), (64, 1030, 4096), (40, 500, 3968), (33, 264, 2000), (200, 4100, 2304), (600, 2048, 512)])
def test_products_of_two_blocks_a_stage(m, n, k):
    """256 columns in a stage, in one part and in several, with ragged last blocks, and an odd number of blocks next to them"""
    test_large_products(m, n, k)


@pytest.mark.parametrize("tile_rows", [5, 16, 32, 48])
@pytest.mark.parametrize("n,k", [(640, 1008), (520, 1152), (300, 2048)])
def test_grouped_product_around_the_ring(tile_rows, n, k):
    """more units than workers, so that the stages' turns run on from one unit into the next"""
    test_grouped_product(tile_rows, 160, 3, 40, n, k, 0)


@pytest.mark.parametrize("m", [1, 12, 17, 40, 90, 200, 300, 777])
@pytest.mark.parametrize("n,k", [(8, 64), (136, 528), (100, 256), (264, 4112), (1032, 2048)])
def test_bf16_rows_are_the_f32_ones_rounded(m, n, k):
    """each output alone takes a way of its own out of the accumulators"""
    import torch
    rng = np.random.default_rng(m + n)
    x, xs, w, ws = codes(rng, m, k), scales(rng, m), codes(rng, n, k), scales(rng, n)
    rc, t = api.i8_upload(w, ws); ok(rc)
    dx, dxs = dev(x), dev(xs)
    y16, z16, y32 = (torch.full((m + 1, n), 3.0, dtype=d, device="cuda") for d in (torch.bfloat16, torch.bfloat16, torch.float32))
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, dx.data_ptr(), 0, dxs.data_ptr(), y16.data_ptr(), 0, here()))
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, dx.data_ptr(), 0, dxs.data_ptr(), z16.data_ptr(), y32.data_ptr(), here()))
    check_product(y16[:m].cpu().view(torch.int16).numpy().view(np.uint16), y32[:m].cpu().numpy(), ref.gemm(x, xs, w, ws))
    assert torch.equal(y16[:m], y32[:m].bfloat16()) and torch.equal(z16, y16) and bool((y16[m] == 3).all())
    api.lib.omega_gpu_i8_free(t)


def test_offsets_past_32_bits():
    """results, rows and codes of more than 2^32 elements: first and last rows of each"""
    import torch
    g = torch.Generator(device="cuda"); g.manual_seed(2)
    m, n, k = 66000, 66000, 64
    x, w = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8, device="cuda") for s in ((m, k), (n, k)))
    xs, ws = torch.rand(m, generator=g, device="cuda") + 0.5, torch.rand(n, generator=g, device="cuda") + 0.5
    rc, t = api.i8_upload_dev(n, k, w.data_ptr(), ws.data_ptr()); ok(rc)
    y = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    ok(api.lib.omega_gpu_i8_gemm_async(t, m, x.data_ptr(), 0, xs.data_ptr(), y.data_ptr(), 0, here()))
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    for rows in (slice(0, 40), slice(32500, 32540), slice(m - 40, m)):
        want = (x[rows].double() @ w.double().T) * torch.outer(xs[rows].double(), ws.double())
        assert bool(((y[rows].double() - want).abs() <= (BF16_HALF * (1 + 2 ** -7) + 4 * EPS24) * want.abs()).all())
    del y, x, w
    api.lib.omega_gpu_i8_free(t)
    T, H = 270000, 16000                                                     # 4.3e9 elements
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q, s = torch.empty((T, H), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    ends = (slice(0, 5), slice(T - 5, T))
    host = [x[r].double().cpu().numpy() for r in ends]
    ok(api.lib.omega_gpu_quant_q8_async(T, H, x.data_ptr(), 1, 0, q.data_ptr(), s.data_ptr(), here()))
    for r, v in zip(ends, host):
        check_rows(q[r].cpu().numpy(), s[r].cpu().numpy(), v, 0.0)
    ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, x.data_ptr(), 0, 0, 0, 0, 0, 0, q.data_ptr(), s.data_ptr(), here()))
    for r, v in zip(ends, host):
        check_rows(q[r].cpu().numpy(), s[r].cpu().numpy(), ref.norm(v, None, 1e-6), 4 * EPS24)


def test_products_on_two_streams_at_once():
    import torch
    rng = np.random.default_rng(11)
    n, k = 512, 1024
    w, ws = codes(rng, n, k), scales(rng, n)
    rc, t = api.i8_upload(w, ws); ok(rc)
    jobs = []
    for m in (1, 20, 130, 700):
        x, xs = codes(rng, m, k), scales(rng, m)
        jobs.append((torch.cuda.Stream(), m, dev(x), dev(xs), torch.zeros((m, n), device="cuda"), ref.gemm(x, xs, w, ws)))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, m, x, xs, y, _ in jobs:
            ok(api.lib.omega_gpu_i8_gemm_async(t, m, x.data_ptr(), 0, xs.data_ptr(), 0, y.data_ptr(), s.cuda_stream))
    torch.cuda.synchronize()
    for _, m, _, _, y, want in jobs:
        assert np.all(np.abs(y.cpu().numpy() - want) <= 3 * EPS24 * np.abs(want))
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    api.lib.omega_gpu_i8_free(t)


def make_plan(ids, E, tile_rows):
    import torch
    T, S = ids.shape
    R = T * S
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")            # noqa: E731
    p = {"ids": dev(ids.astype(np.uint32)), "counts": z(E), "starts": z(E), "xmap": z(R + 8), "ymap": z(R + 8), "tiles": z(4 * (R + E)), "header": z(8), "most": R // tile_rows + min(E, R)}
    o = api.MoePlanOut(p["counts"].data_ptr(), p["starts"].data_ptr(), p["xmap"].data_ptr(), p["ymap"].data_ptr(), 0, 0, 0, 0, p["tiles"].data_ptr(), p["header"].data_ptr())
    ok(api.lib.omega_gpu_moe_plan_async(C.c_uint32(T), C.c_uint32(S), C.c_uint32(E), C.c_uint32(S), C.c_uint32(tile_rows), C.c_uint64(p["ids"].data_ptr()), C.byref(o), C.c_void_p(here())))
    return p


@pytest.mark.parametrize("tile_rows", [1, 8, 16, 32, 100, 128, 256])
@pytest.mark.parametrize("T,S,E,n,k,skew", [(1, 4, 6, 64, 64, 0), (21, 3, 10, 100, 208, 0), (64, 4, 8, 272, 512, 1), (300, 2, 3, 128, 96, 0)])
def test_grouped_product(tile_rows, T, S, E, n, k, skew):
    import torch
    rng = np.random.default_rng(T + tile_rows)
    pool = np.arange(E) if not skew else np.arange(S)                         # skewed: most experts stay empty
    ids = np.stack([rng.choice(pool, S, replace=False) for _ in range(T)])
    ids[T // 2, 0] = ids[T // 2, 0] if T == 1 else -1                         # an absent pick
    R = T * S
    x, xs, w, ws = codes(rng, T, k), scales(rng, T), codes(rng, E * n, k), scales(rng, E * n)
    rc, t = api.i8_upload(w, ws); ok(rc)
    p, dx, dxs = make_plan(ids, E, tile_rows), dev(x), dev(xs)
    y16, y32 = torch.full((R, n), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((R, n), 3.0, device="cuda")
    args = lambda xm, ym, a, b, rows, sc: (t, E, tile_rows, p["most"], p["tiles"].data_ptr(), p["header"].data_ptr(), xm, ym, a, rows, b, y16.data_ptr(), y32.data_ptr(), here())   # noqa: E731
    ok(api.lib.omega_gpu_i8_gemm_grouped_async(*args(p["xmap"].data_ptr(), p["ymap"].data_ptr(), dx.data_ptr(), dxs.data_ptr(), T, dxs)))
    flat = ids.reshape(-1)
    want = np.stack([ref.gemm(x[i // S:i // S + 1], xs[i // S:i // S + 1], w[e * n:(e + 1) * n], ws[e * n:(e + 1) * n])[0] if e >= 0 else np.full(n, 3.0) for i, e in enumerate(flat)])
    check_product(y16.cpu().view(torch.int16).numpy().view(np.uint16), y32.cpu().numpy(), want)
    # without maps: sorted rows in, sorted rows out
    order = np.argsort(np.where(flat < 0, E, flat), kind="stable")[:(flat >= 0).sum()]
    xo, so = dev(x[order // S]), dev(xs[order // S])
    y16.fill_(3.0); y32.fill_(3.0)
    ok(api.lib.omega_gpu_i8_gemm_grouped_async(*args(0, 0, xo.data_ptr(), so.data_ptr(), len(order), so)))
    got = y32.cpu().numpy()
    check_product(y16.cpu().view(torch.int16).numpy().view(np.uint16)[:len(order)], got[:len(order)], want[order])
    assert (got[len(order):] == 3).all()
    # bf16 rows alone, with and without maps
    z16 = torch.full((R, n), 3.0, dtype=torch.bfloat16, device="cuda")
    for xm, ym, a, b, rows, f32 in ((0, 0, xo, so, len(order), y32), (p["xmap"].data_ptr(), p["ymap"].data_ptr(), dx, dxs, T, dev(np.where(np.isnan(want), 0, want).astype(np.float32)))):
        z16.fill_(3.0)
        ok(api.lib.omega_gpu_i8_gemm_grouped_async(t, E, tile_rows, p["most"], p["tiles"].data_ptr(), p["header"].data_ptr(), xm, ym, a.data_ptr(), rows, b.data_ptr(), z16.data_ptr(), 0, here()))
        near = (z16.float() - f32).abs() <= (BF16_HALF * (1 + 2 ** -7) + 4 * EPS24) * f32.abs()
        assert bool(near.all())
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    api.lib.omega_gpu_i8_free(t)


@pytest.mark.parametrize("tile_rows", [16, 48, 160])
@pytest.mark.parametrize("gathered", [True, False])
def test_grouped_product_of_a_plan_of_ones_own(tile_rows, gathered):
    """tiles in any order, experts twice, tiles without rows, at the first place and the last one too"""
    import torch
    rng = np.random.default_rng(tile_rows)
    E, n, k, R = 5, 264, 640, 400
    counts = [0, tile_rows, 3, 0, 0, 17 % tile_rows, tile_rows - 1, 1, 0]
    experts = [2, 4, 0, 1, 4, 4, 3, 0, 3]
    rows = np.cumsum([0] + counts[:-1])
    tiles = np.zeros((len(counts) + 3, 4), np.uint32)
    tiles[:len(counts), 0], tiles[:len(counts), 1], tiles[:len(counts), 2] = experts, rows, counts
    total = int(sum(counts)); assert total <= R
    x, xs, w, ws = codes(rng, R, k), scales(rng, R), codes(rng, E * n, k), scales(rng, E * n)
    xmap, ymap = rng.integers(0, R, total).astype(np.uint32), rng.permutation(R)[:total].astype(np.uint32)
    rc, t = api.i8_upload(w, ws); ok(rc)
    y, dt, dh = torch.full((R, n), 3.0, device="cuda"), dev(tiles), dev(np.array([0, 0, len(counts), 0], np.uint32))
    dx, dxs, dxm, dym = dev(x), dev(xs), dev(xmap), dev(ymap)
    ok(api.lib.omega_gpu_i8_gemm_grouped_async(t, E, tile_rows, len(tiles), dt.data_ptr(), dh.data_ptr(), dxm.data_ptr() if gathered else 0, dym.data_ptr(), dx.data_ptr(), R, dxs.data_ptr(), 0, y.data_ptr(), here()))
    assert api.lib.omega_gpu_i8_status(t, here()) == 0
    want = np.full((R, n), 3.0)
    for e, r0, c in zip(experts, rows, counts):
        for r in range(r0, r0 + c):
            src = xmap[r] if gathered else r
            want[ymap[r]] = ref.gemm(x[src:src + 1], xs[src:src + 1], w[e * n:(e + 1) * n], ws[e * n:(e + 1) * n])[0]
    assert np.all(np.abs(y.cpu().numpy() - want) <= 3 * EPS24 * np.abs(want))
    api.lib.omega_gpu_i8_free(t)


def test_grouped_product_after_a_refused_plan_does_nothing():
    import torch
    rng = np.random.default_rng(1)
    E, n, k = 4, 64, 64
    rc, t = api.i8_upload(codes(rng, E * n, k), scales(rng, E * n)); ok(rc)
    p, dx, dxs = make_plan(np.array([[0, 9]]), E, 16), dev(codes(rng, 1, k)), dev(scales(rng, 1))
    y = torch.full((2, n), 3.0, device="cuda")
    ok(api.lib.omega_gpu_i8_gemm_grouped_async(t, E, 16, p["most"], p["tiles"].data_ptr(), p["header"].data_ptr(), p["xmap"].data_ptr(), p["ymap"].data_ptr(), dx.data_ptr(), 1, dxs.data_ptr(), 0,
                                               y.data_ptr(), here()))
    assert (y == 3).all() and p["header"][3] == 2
    api.lib.omega_gpu_i8_free(t)


# ------------------------------------------------------------------ the layer, and norm and layer together
class Layer:
    def __init__(self, seed, E, H, I, K, most, sigmoid=True, groups=1, kept=0, rank=1, biased=True):
        rng = np.random.default_rng(seed)
        self.gu, self.gus, self.dn, self.dns = codes(rng, E, 2 * I, H), scales(rng, (E, 2 * I), 0.0005), codes(rng, E, H, I), scales(rng, (E, H), 0.0005)
        self.bias = rng.normal(0, 0.1, E).astype(np.float32) if biased else None
        self.how = dict(topk=K, sigmoid=sigmoid, bias=self.bias, groups=groups, kept=kept, rank=rank)
        rc, self.tgu = api.i8_upload(self.gu.reshape(-1, H), self.gus.reshape(-1)); ok(rc)
        rc, self.tdn = api.i8_upload(self.dn.reshape(-1, I), self.dns.reshape(-1)); ok(rc)
        rc, self.h = api.moe_i8_layer_create(self.tgu, self.tdn, config(E, K, sigmoid, groups, kept, rank), self.bias, most); ok(rc)

    def want(self, logits_bits, q, s):
        ids, w = ref.route(api.bf16_to_f32(logits_bits), **self.how)
        return ids, w, ref.layer(ids, w, q.astype(np.float64), s.astype(np.float64), self.gu, self.gus, self.dn, self.dns)

    def free(self):
        api.lib.omega_gpu_moe_i8_layer_free(self.h); api.lib.omega_gpu_i8_free(self.tgu); api.lib.omega_gpu_i8_free(self.tdn)


def quantised(x_bits):
    import torch
    T, H = x_bits.shape
    d, q, s = dev(x_bits), torch.zeros((T, H), dtype=torch.int8, device="cuda"), torch.zeros(T, device="cuda")
    ok(api.lib.omega_gpu_quant_q8_async(T, H, d.data_ptr(), 1, 0, q.data_ptr(), s.data_ptr(), here()))
    return q.cpu().numpy(), s.cpu().numpy()


# Of the codes between the two products, those next to a border may come out one off: 127 * 2 * GATE_REL(8) of them at most, and those whose gate|up value lies next to a border
# of bf16 (4 * EPS24 * 2^8 of each of the two). One code off is 1/30 of a code's rms (codes of such rows have an rms of 30 or so), so the relative 2-norm of the
# difference is sqrt(127 * 2 * 2e-6 + 1.3e-4) / 30 = 8.4e-4 where all of them fall the other way.
LAYER_REL = 1e-3


@pytest.mark.parametrize("T", [1, 3, 40, 260])
@pytest.mark.parametrize("E,H,I,K,groups,kept,rank", [(8, 256, 128, 2, 1, 0, 1), (16, 528, 208, 4, 4, 2, 2), (6, 1024, 272, 3, 1, 0, 1)])
def test_layer(T, E, H, I, K, groups, kept, rank):
    L = Layer(T + E, E, H, I, K, T, groups=groups, kept=kept, rank=rank, sigmoid=E != 6, biased=E != 6)
    rng = np.random.default_rng(T)
    lg, x = bits(rng.normal(0, 1, (T, E)).astype(np.float32)), bits(rng.normal(0, 1, (T, H)).astype(np.float32))
    rc, o16, o32, ids, w = api.moe_i8_layer_bf16(L.h, lg, x, K); ok(rc)
    # bf16 rows hit the borders between two codes exactly (254 x / largest is an odd number), and either code is right there: the codes are the library's own, checked
    q, s = quantised(x)
    check_rows(q, s, api.bf16_to_f32(x).astype(np.float64), 0.0)
    wids, ww, want = L.want(lg, q, s)
    assert np.array_equal(ids, wids) and np.all(np.abs(w - ww) <= (K + 5) * EPS24 * ww)
    assert np.linalg.norm(o32 - want) <= LAYER_REL * np.linalg.norm(want)
    assert np.all(np.abs(api.bf16_to_f32(o16) - o32) <= BF16_HALF * np.abs(o32))
    assert api.lib.omega_gpu_moe_i8_layer_status(L.h, here()) == 0
    assert api.lib.omega_gpu_moe_i8_layer_launches(L.h) == (6 if T == 1 else 7 + (T * K // E >= 65))     # one token needs no plan; many rows are sorted first
    # fewer tokens than the layer has room for: the same rows
    if T > 3:
        rc, _, p32, _, _ = api.moe_i8_layer_bf16(L.h, lg[1:4], x[1:4], K); ok(rc)
        assert np.array_equal(p32.view(np.uint32), o32[1:4].view(np.uint32))
    L.free()


def test_norm_and_layers_in_a_row():
    """two layers on a residual stream, as a decode loop runs them: norm to 8-bit rows, layer, norm with the layer's rows added, layer, last addition"""
    import torch
    T, E, H, I, K = 37, 16, 512, 256, 4
    L = [Layer(i, E, H, I, K, T, groups=4, kept=2, rank=2) for i in (1, 2)]
    rng = np.random.default_rng(9)
    x = bits(rng.normal(0, 1, (T, H)).astype(np.float32)); lg = [bits(rng.normal(0, 1, (T, E)).astype(np.float32)) for _ in L]; nw = [rng.normal(1, 0.1, H).astype(np.float32) for _ in L]
    s = torch.cuda.Stream()
    dx, dl, dn = dev(x), [dev(v) for v in lg], [dev(v) for v in nw]
    h, m, q, sc, last = torch.zeros((T, H), device="cuda"), torch.zeros((T, H), device="cuda"), torch.zeros((T, H), dtype=torch.int8, device="cuda"), torch.zeros(T, device="cuda"), torch.zeros((T, H), device="cuda")
    torch.cuda.synchronize()
    seen = []
    for i in (0, 1):
        ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, 0 if i else dx.data_ptr(), m.data_ptr() if i else 0, 0, h.data_ptr() if i else 0, h.data_ptr(), dn[i].data_ptr(), 0, q.data_ptr(), sc.data_ptr(), s.cuda_stream))
        with torch.cuda.stream(s):
            seen.append((h.clone(), q.clone(), sc.clone()))
        ok(api.lib.omega_gpu_moe_i8_layer_q8_async(L[i].h, T, dl[i].data_ptr(), q.data_ptr(), sc.data_ptr(), m.data_ptr(), 0, s.cuda_stream))
        with torch.cuda.stream(s):
            seen[i] += (m.clone(),)
    with torch.cuda.stream(s):
        last = h + m
    s.synchronize()
    at = api.bf16_to_f32(x)
    for i in (0, 1):
        gh, gq, gs, gm = (v.cpu().numpy() for v in seen[i])
        assert np.array_equal(gh, at)                                        # f32 additions, the same here
        check_rows(gq, gs, ref.norm(gh.astype(np.float64), nw[i], 1e-6), 4 * EPS24)
        _, _, want = L[i].want(lg[i], gq, gs)
        assert np.linalg.norm(gm - want) <= LAYER_REL * np.linalg.norm(want)
        at = at + gm
    assert np.array_equal(last.cpu().numpy(), at)
    for l in L:
        l.free()


def test_route_feeds_the_fp8_layer():
    """ids and weights of the new routing through omega_gpu_moe_layer_routed_async: softmax without bias or groups picks what that layer's own top-k picks"""
    import torch
    from tests.test_gpu_layer import build_layer, free_layer
    E, H, I, T, K = 16, 512, 256, 40, 4
    m = build_layer(np.random.default_rng(4), E, H, I, T, api.ENGINE_MMA, K)
    g = torch.Generator(device="cuda"); g.manual_seed(3)
    lg, x = torch.randn((T, E), generator=g, device="cuda").bfloat16(), torch.randn((T, H), generator=g, device="cuda").bfloat16()
    ids, w, a, b = torch.zeros((T, K), dtype=torch.int32, device="cuda"), torch.zeros((T, K), device="cuda"), torch.zeros((T, H), device="cuda"), torch.zeros((T, H), device="cuda")
    V = C.c_uint64
    ok(api.lib.omega_gpu_moe_layer_async(m["layer"], C.c_uint32(T), V(lg.data_ptr()), V(x.data_ptr()), V(a.data_ptr()), V(0), C.c_void_p(here())))
    ok(api.lib.omega_gpu_moe_route_async(config(E, K, False), T, lg.data_ptr(), 1, 0, 0, ids.data_ptr(), w.data_ptr(), here()))
    ok(api.lib.omega_gpu_moe_layer_routed_async(m["layer"], C.c_uint32(T), V(ids.data_ptr()), V(w.data_ptr()), V(x.data_ptr()), V(b.data_ptr()), V(0), C.c_void_p(here())))
    torch.cuda.synchronize()
    assert float((a - b).norm() / a.norm()) <= 20 * EPS24                     # the same rows under weights that differ by a few roundings
    free_layer(m)


# ------------------------------------------------------------------ captured calls
def test_captured_calls():
    import torch
    from tests.test_gpu_capture import compare
    T, E, H, I, K = 24, 16, 512, 256, 4
    L = Layer(5, E, H, I, K, T, groups=4, kept=2, rank=2)
    lg, x = torch.zeros((T, E), dtype=torch.bfloat16, device="cuda"), torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    q, s, o32, o16 = torch.zeros((T, H), dtype=torch.int8, device="cuda"), torch.zeros(T, device="cuda"), torch.zeros((T, H), device="cuda"), torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")

    def fill(inputs, seed):
        g = torch.Generator(device="cuda"); g.manual_seed(seed)
        for t in inputs:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))

    def call():
        ok(api.lib.omega_gpu_residual_norm_q8_async(T, H, 1e-6, x.data_ptr(), 0, 0, 0, 0, 0, 0, q.data_ptr(), s.data_ptr(), here()))
        ok(api.lib.omega_gpu_moe_i8_layer_q8_async(L.h, T, lg.data_ptr(), q.data_ptr(), s.data_ptr(), o32.data_ptr(), o16.data_ptr(), here()))
        return o32, o16
    compare(call, [lg, x], fill, torch.zeros(4, device="cuda"))
    L.free()


@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_product(m):
    import torch
    from tests.test_gpu_capture import compare
    rng = np.random.default_rng(m)
    n, k = 384, 1024
    rc, t = api.i8_upload(codes(rng, n, k), scales(rng, n)); ok(rc)
    x, q, s, y = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda"), torch.zeros((m, k), dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda"), torch.zeros((m, n), device="cuda")

    def fill(inputs, seed):
        g = torch.Generator(device="cuda"); g.manual_seed(seed)
        inputs[0].copy_(torch.randn(x.shape, generator=g, device="cuda"))

    def call():
        ok(api.lib.omega_gpu_quant_q8_async(m, k, x.data_ptr(), 1, 0, q.data_ptr(), s.data_ptr(), here()))
        ok(api.lib.omega_gpu_i8_gemm_async(t, m, q.data_ptr(), 0, s.data_ptr(), 0, y.data_ptr(), here()))
        return (y,)
    compare(call, [x], fill, torch.zeros(4, device="cuda"))
    api.lib.omega_gpu_i8_free(t)
