"""Layers called with one token count after another, as a prefill in chunks does: every result is that of a layer which has seen no other call. From 4096 picks on the routing
plan is made by three launches that share a scratch over calls of any size."""
import ctypes as C

import numpy as np
import pytest

from cudapp_b200 import api
from oracle import oracle as orc

pytestmark = pytest.mark.gpu
U32 = C.c_uint32
SIZES = (4096, 1500, 2048, 600, 513, 1024, 3000, 1, 4096)


def same_as_fresh_layers(make, run, free, E, H):
    rng = np.random.default_rng(E + H)
    most = max(SIZES)
    logits = orc.bf16_bits((rng.normal(0, 1, (most, E)) + rng.normal(0, 0.5, E)).astype(np.float32)); x = orc.bf16_bits(rng.normal(0, 1, (most, H)).astype(np.float32))
    layer = make(most)
    for i, tokens in enumerate(SIZES):
        order = rng.permutation(most)[:tokens]                             # other tokens in every call: nothing left over can pass for a result
        lg, xb = np.ascontiguousarray(logits[order]), np.ascontiguousarray(x[order])
        fresh = make(tokens)
        got, want = run(layer, lg, xb), run(fresh, lg, xb)
        free(fresh)
        for a, b in zip(got, want):
            assert np.array_equal(a.view(np.uint32 if a.itemsize == 4 else np.uint16), b.view(np.uint32 if b.itemsize == 4 else np.uint16)), (i, tokens)
        assert np.any(got[0])
    free(layer)


def test_8_bit_integer_layer():
    from tests.test_gpu_i8 import codes, config, ok, scales
    rng = np.random.default_rng(1)
    E, H, I, K = 128, 256, 128, 8
    rc, gu = api.i8_upload(codes(rng, E * 2 * I, H), scales(rng, E * 2 * I, 0.0005)); ok(rc)
    rc, dn = api.i8_upload(codes(rng, E * H, I), scales(rng, E * H, 0.0005)); ok(rc)

    def make(tokens):
        rc, h = api.moe_i8_layer_create(gu, dn, config(E, K, True, 8, 4, 2), None, tokens); ok(rc)
        return h

    def run(h, lg, x):
        rc, o16, o32, ids, w = api.moe_i8_layer_bf16(h, lg, x, K); ok(rc)
        return o32.copy(), o16.copy(), ids, w
    same_as_fresh_layers(make, run, api.lib.omega_gpu_moe_i8_layer_free, E, H)
    api.lib.omega_gpu_i8_free(gu); api.lib.omega_gpu_i8_free(dn)


@pytest.mark.parametrize("engine,pieces", [(api.ENGINE_MMA, (2, 3)), (api.ENGINE_MMA, (1, 1)), (api.ENGINE_FMA, (2, 3))])
def test_fp8_layer(engine, pieces):
    from tests.test_gpu_layer import build_layer, free_layer
    E, H, I, K = 128, 512, 256, 8
    m = build_layer(np.random.default_rng(2), E, H, I, 8, engine, K)

    def make(tokens):
        rc, h = api.moe_layer_create(m["tgu"], m["tdn"], topk=K, max_tokens=tokens, engine=engine, x_pieces=pieces[0], act_pieces=pieces[1]); assert rc == 0, api.last_error()
        return h

    def run(h, lg, x):
        rc, o16, o32, ids, w = api.moe_layer_bf16(h, lg, x, K); assert rc == 0, api.last_error()
        return o32.copy(), o16.copy(), ids, w
    same_as_fresh_layers(make, run, api.lib.omega_gpu_moe_layer_free, E, H)
    free_layer(m)


def test_4_bit_layer():
    rng = np.random.default_rng(3)
    E, H, I, K = 128, 768, 768, 8

    def tensor(n, k):
        t = C.c_void_p(); packed = rng.integers(0, 256, (n, k // 2), dtype=np.uint8); scale = rng.integers(118, 122, (n, k // 32), dtype=np.uint8)
        assert api.lib.omega_gpu_mxfp4_upload(U32(n), U32(k), api._p(packed), api._p(scale), C.byref(t)) == 0, api.last_error()
        return t
    gu, dn = tensor(E * 2 * I, H), tensor(E * H, I)

    def make(tokens):
        h = C.c_void_p()
        assert api.lib.omega_gpu_moe_w4_layer_create(gu, dn, U32(E), U32(K), U32(tokens), C.c_int(1), C.byref(h)) == 0, api.last_error()
        return h

    def run(h, lg, x):
        out, ids = np.zeros(x.shape, np.float32), np.zeros((len(x), K), np.uint32)
        assert api.lib.omega_gpu_moe_w4_layer_bf16(h, U32(len(x)), api._p(lg), api._p(x), None, api._p(out), api._p(ids), None) == 0, api.last_error()
        return out, ids
    same_as_fresh_layers(make, run, api.lib.omega_gpu_moe_w4_layer_free, E, H)
    api.lib.omega_gpu_w4_free(gu); api.lib.omega_gpu_w4_free(dn)


class I8Layer(C.Structure):
    """the 8-bit integer layer's own record, up to the plan's scratch"""
    _fields_ = ([(n, C.c_void_p) for n in ("gu", "dn")] + [("route", api.MoeRouteConfig)] + [(n, U32) for n in ("hidden", "inter", "max_tokens", "launches")] +
                [(n, C.c_void_p) for n in ("base", "bias", "wts", "xs", "ss", "as_", "out32", "xq", "sq", "aq", "logits", "x", "gu16", "dn16", "out16", "ids", "counts", "starts", "xmap", "ymap",
                                           "tiles", "header", "scratch")])


class Refusable:
    """a layer whose next plan can be made to refuse: the word that says an id was out of range is set beforehand"""

    def __init__(self, most):
        from tests.test_gpu_i8 import codes, config, ok, scales
        rng = np.random.default_rng(4)
        self.E, self.H, self.I, self.K = 8, 256, 128, 8
        rc, self.gu = api.i8_upload(codes(rng, self.E * 2 * self.I, self.H), scales(rng, self.E * 2 * self.I, 0.0005)); ok(rc)
        rc, self.dn = api.i8_upload(codes(rng, self.E * self.H, self.I), scales(rng, self.E * self.H, 0.0005)); ok(rc)
        rc, self.h = api.moe_i8_layer_create(self.gu, self.dn, config(self.E, self.K, True), None, most); ok(rc)
        self.own = C.cast(self.h, C.POINTER(I8Layer)).contents
        assert (self.own.hidden, self.own.inter, self.own.max_tokens) == (self.H, self.I, most)

    def inputs(self, tokens):
        rng = np.random.default_rng(tokens)
        return orc.bf16_bits(rng.normal(0, 1, (tokens, self.E)).astype(np.float32)), orc.bf16_bits(rng.normal(0, 1, (tokens, self.H)).astype(np.float32))

    def copy(self, dst, src, nbytes):
        import torch
        torch.cuda.synchronize()
        assert C.CDLL("libcudart.so.12").cudaMemcpy(C.c_void_p(dst), C.c_void_p(src), C.c_size_t(nbytes), 4) == 0     # 4: either way

    def refuse_next(self):
        word = np.ones(1, np.uint32)
        self.copy(self.own.scratch, word.ctypes.data, 4)

    def read(self, at, shape, dtype):
        out = np.zeros(shape, dtype)
        self.copy(out.ctypes.data, at, out.nbytes)
        return out

    def free(self):
        api.lib.omega_gpu_moe_i8_layer_free(self.h); api.lib.omega_gpu_i8_free(self.gu); api.lib.omega_gpu_i8_free(self.dn)


def test_a_refused_plan_moves_no_rows():
    """the maps are then those of the call before, whose rows may lie past this call's"""
    import torch
    from tests.test_gpu_i8 import dev, here, ok
    m = Refusable(1024)
    out = torch.zeros((1024, m.H), device="cuda")

    def call(tokens):
        lg, x = (dev(v) for v in m.inputs(tokens))
        ok(api.lib.omega_gpu_moe_i8_layer_async(m.h, tokens, lg.data_ptr(), x.data_ptr(), out.data_ptr(), 0, here()))
        torch.cuda.synchronize()
        return out[:tokens].clone()
    call(1024)
    before = m.read(m.own.sq, (1024 * m.K, m.H), np.int8), m.read(m.own.ss, 1024 * m.K, np.float32)
    m.refuse_next()
    call(600)
    header = m.read(m.own.header, 4, np.uint32)
    assert list(header) == [0, 0, 0, 2]
    after = m.read(m.own.sq, (1024 * m.K, m.H), np.int8), m.read(m.own.ss, 1024 * m.K, np.float32)
    assert all(np.array_equal(a, b) for a, b in zip(before, after))
    first = call(600)                                                      # the word is clear again
    assert list(m.read(m.own.header, 4, np.uint32))[3] == 0 and torch.equal(call(600), first)
    assert not np.array_equal(m.read(m.own.sq, (1024 * m.K, m.H), np.int8), before[0])
    m.free()


def test_a_refused_plan_is_reported():
    import torch
    from tests.test_gpu_i8 import dev, here, ok
    m = Refusable(600)
    lg, x = m.inputs(600)
    rc, _, want, _, _ = api.moe_i8_layer_bf16(m.h, lg, x, m.K); ok(rc)
    want = want.copy()
    m.refuse_next()
    rc, _, _, _, _ = api.moe_i8_layer_bf16(m.h, lg, x, m.K)
    assert rc == api.BAD_ARGS and "refused (status 2)" in api.last_error()
    m.refuse_next()
    dl, dx, out = dev(lg), dev(x), torch.zeros((600, m.H), device="cuda")
    ok(api.lib.omega_gpu_moe_i8_layer_async(m.h, 600, dl.data_ptr(), dx.data_ptr(), out.data_ptr(), 0, here()))
    assert api.lib.omega_gpu_moe_i8_layer_status(m.h, here()) == 102
    for tokens in (600, 1):                                                # nothing of it stays
        rc, _, got, _, _ = api.moe_i8_layer_bf16(m.h, lg[:tokens], x[:tokens], m.K); ok(rc)
        assert np.array_equal(got.view(np.uint32), want[:tokens].view(np.uint32)) and api.lib.omega_gpu_moe_i8_layer_status(m.h, here()) == 0
    m.free()


@pytest.mark.parametrize("E,T", [(5, 9), (700, 40)])
def test_a_refused_plan_has_no_segments(E, T):
    """records of the plan before would be taken for its own by a product that walks them"""
    import torch
    rng = np.random.default_rng(E)
    S, R = 3, T * 3
    ids = rng.integers(0, E, (T, S)).astype(np.int32)
    z = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device="cuda")     # noqa: E731
    counts, starts, xmap, ymap, seg_a, seg_b, header = z(E), z(E), z(R + 8), z(R + 8), z(8 * E), z(8 * E), z(8)
    table = torch.arange(16, 16 + 2 * E, device="cuda")
    o = api.MoePlanOut(counts.data_ptr(), starts.data_ptr(), xmap.data_ptr(), ymap.data_ptr(), seg_a.data_ptr(), table.data_ptr(), seg_b.data_ptr(), table.data_ptr(), 0, header.data_ptr())

    def plan(v):
        d = torch.from_numpy(v).cuda()
        rc = api.lib.omega_gpu_moe_plan_async(U32(T), U32(S), U32(E), U32(S), U32(0), C.c_uint64(d.data_ptr()), C.byref(o), C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0, api.last_error()
        torch.cuda.synchronize()
    assert api.lib.omega_gpu_moe_topk_bf16(U32(1), U32(1), U32(1), C.c_int(1), api._p(np.zeros(1, np.uint16)), api._p(np.zeros(1, np.uint32)), api._p(np.zeros(1, np.float32))) == 0   # opens the device
    plan(ids)
    assert header[3] == 0 and int((seg_a.view(E, 8)[:, 5] > 0).sum()) == len(np.unique(ids)) and torch.equal(seg_a, seg_b)
    kept = [t.clone() for t in (counts, starts, xmap, ymap)]
    bad = ids.copy(); bad[T // 2, 1] = E
    plan(bad)
    assert header[:4].tolist() == [0, 0, 0, 2] and not seg_a.any() and not seg_b.any()
    assert all(torch.equal(a, b) for a, b in zip(kept, (counts, starts, xmap, ymap)))


def test_fp8_layer_on_the_exact_engine_after_a_refused_plan():
    """a call of 2 tokens with an id outside the layer, after one of 64: nothing is read through the 64 tokens' maps, and the next call is right"""
    import torch
    from tests.test_gpu_layer import build_layer, free_layer
    E, H, I, K = 8, 512, 256, 2
    m = build_layer(np.random.default_rng(6), E, H, I, 64, api.ENGINE_FMA, K)
    g = torch.Generator(device="cuda"); g.manual_seed(1)
    x, w, out = torch.randn((64, H), generator=g, device="cuda").bfloat16(), torch.rand((64, K), generator=g, device="cuda"), torch.zeros((64, H), device="cuda")
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i))[:K] for i in range(64)]).int().cuda()
    s, V = C.c_void_p(torch.cuda.current_stream().cuda_stream), lambda t: C.c_uint64(t.data_ptr())

    def call(n, ids):
        xs = x[:n].clone()
        rc = api.lib.omega_gpu_moe_layer_routed_async(m["layer"], U32(n), V(ids), V(w), V(xs), V(out), C.c_uint64(0), s); assert rc == 0, api.last_error()
        return api.lib.omega_gpu_moe_layer_status(m["layer"], s)
    assert call(64, ids) == 0
    want = out.clone()
    bad = ids[:2].clone(); bad[1, 0] = E
    assert call(2, bad) == 102
    assert call(2, ids) == 0 and torch.equal(out[:2], want[:2])
    assert call(64, ids) == 0 and torch.equal(out, want)
    free_layer(m)
