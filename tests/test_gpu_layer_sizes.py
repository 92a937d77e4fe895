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
