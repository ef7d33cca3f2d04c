"""GPU tests of the layer steps over a bounded cache: equal to the plain layer steps, bit for bit, where
the row is the position; the appended rows the same wherever they go; the weights against float64 over
the step's own queries (tolerance: test_evict_gpu.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import to_dev
from test_evict_gpu import D, H, KV, attend64, check, f16_cache, gen, randn, weights64
from test_layer_gpu import q4k_blocks, q6k_blocks

pytestmark = pytest.mark.gpu

EPS = 1e-6


def make_layer(O, attn, q_format):
    rng = np.random.default_rng(5)
    q4 = lambda n, k: (to_dev(torch, O.q4k_repack_r1(q4k_blocks(rng, n, k))), "q4_k")  # noqa: E731
    q6 = lambda n, k: (to_dev(torch, O.q6k_repack_r1(q6k_blocks(rng, n, k), n, k)), "q6_k")  # noqa: E731
    norms = [to_dev(torch, (1 + 0.1 * rng.standard_normal(n)).astype(np.float32))
             for n in (2048, 256, 256)]
    q = q4(8192, 2048) if q_format == "q4_k" else q6(8192, 2048)
    return attn.Layer(q, q4(512, 2048), q6(512, 2048), q4(2048, 4096), *norms,
                      to_dev(torch, O.inv_freq(1e7)))


@pytest.fixture(scope="module")
def layers(O, attn):
    return {f: make_layer(O, attn, f) for f in ("q4_k", "q6_k")}


def decode_queries(attn, ws):
    at = int(attn._lib.load().miso_attn_layer_decode_core()) - H * D  # q lies before the core
    return ws.decode[at:at + H * D].view(1, H, D).clone()


def prefill_queries(attn, ws, n):
    at = int(attn._lib.load().miso_attn_layer_prefill_core(ws.max_tok)) - ws.max_tok * H * D
    return ws.prefill[at:at + n * H * D].view(n, H, D).clone()


@pytest.mark.parametrize("fmt", ["q4_k", "q6_k"])
@pytest.mark.parametrize("row", [0, 1, 5, 40, 300, 3001])
@pytest.mark.parametrize("with_delta", [True, False])
def test_layer_decode_weights(attn, layers, fmt, row, with_delta):
    g = gen(row + 1)
    ctx = row + 9
    k, v = f16_cache(g, row, ctx)
    h, delta = randn(g, 2048), 0.3 * randn(g, 2048) if with_delta else None
    ws, sc = attn.LayerWorkspace(max_tok=16), attn.DecodeWeightsScratch(attn.LAYER_MAX_SPLITS, ctx)
    before = torch.rand(KV, ctx, generator=g, device="cuda") / (row + 1)
    w = before.clone()
    got = [t.clone() for t in (h, k, v)]
    y, y0 = torch.empty(2048, device="cuda"), torch.empty(2048, device="cuda")
    attn.layer_decode_weights(layers[fmt], got[1], got[2], ctx, row, row, got[0], delta, y, EPS, ws,
                              w, sc)
    q = decode_queries(attn, ws)
    attn.layer_decode(layers[fmt], k, v, ctx, row, h, delta, y0, EPS, ws)
    assert torch.equal(y, y0)
    for a, b in zip(got, (h, k, v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    added, rel = weights64(q, k[:, :row + 1].double(), row)
    check(w[:, :row + 1], before[:, :row + 1], added, rel)
    assert torch.equal(w[:, row + 1:], before[:, row + 1:])


@pytest.mark.parametrize("fmt", ["q4_k", "q6_k"])
@pytest.mark.parametrize("row,pos", [(0, 17), (60, 400), (400, 60), (2000, 9000)])
def test_layer_decode_weights_at_another_row(attn, layers, fmt, row, pos):
    g = gen(row + pos)
    ctx, big = row + 4, pos + 4
    k, v = f16_cache(g, row, ctx)
    old = [k.clone(), v.clone()]
    kb, vb = f16_cache(g, pos, big)
    h = randn(g, 2048)
    ws, sc = attn.LayerWorkspace(max_tok=16), attn.DecodeWeightsScratch(attn.LAYER_MAX_SPLITS, ctx)
    w, y = torch.zeros(KV, ctx, device="cuda"), torch.empty(2048, device="cuda")
    attn.layer_decode(layers[fmt], kb, vb, big, pos, h.clone(), None, y, EPS, ws)
    attn.layer_decode_weights(layers[fmt], k, v, ctx, row, pos, h, None, y, EPS, ws, w, sc)
    q, core = decode_queries(attn, ws), ws.decode_core.view(1, H, D).clone()
    at = int(attn._lib.load().miso_attn_layer_decode_core()) - H * D - 9216
    qg = ws.decode[at:at + 8192].view(1, H, 2, D)
    for a, b, c in ((k, kb, old[0]), (v, vb, old[1])):
        # the row may be prepared in the split's workgroup or by the prep's kernel (row 0)
        assert torch.allclose(a[:, row].float(), b[:, pos].float(), rtol=2 ** -9, atol=1e-3)
        a[:, row] = c[:, row]
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    attn.layer_decode_weights(layers[fmt], k, v, ctx, row, pos, h, None, y, EPS, ws,
                              torch.zeros_like(w), sc)
    k64, v64 = (t[:, :row + 1].double() for t in (k, v))
    added, rel = weights64(q, k64, row)
    check(w[:, :row + 1], torch.zeros_like(w[:, :row + 1]), added, rel)
    want = attend64(q, qg, k64, v64, row)
    for i in range(H):  # the reference's gate for a decode
        assert float((core[0, i].double() - want[0, i]).norm() / want[0, i].norm()) <= 1e-5


@pytest.mark.parametrize("row0,n", [(0, 1), (0, 16), (33, 40), (700, 129)])
@pytest.mark.parametrize("voters", [None, 0, 7])
def test_layer_prefill_weights(attn, layers, row0, n, voters):
    g = gen(row0 + n)
    rows = row0 + n
    ctx = rows + 5
    k, v = f16_cache(g, row0, ctx)
    h, delta = randn(g, n * 2048), 0.3 * randn(g, n * 2048)
    ws, sc = attn.LayerWorkspace(max_tok=160), attn.PrefillWeightsScratch(n, rows)
    before = torch.rand(KV, ctx, generator=g, device="cuda")
    w = before.clone()
    got = [t.clone() for t in (h, k, v)]
    y, y0 = (torch.empty(n * 2048, device="cuda") for _ in range(2))
    attn.layer_prefill_weights(layers["q4_k"], got[1], got[2], ctx, row0, row0, n, got[0], delta, y,
                               EPS, ws, w, sc, voters=voters)
    q = prefill_queries(attn, ws, n)
    attn.layer_prefill(layers["q4_k"], k, v, ctx, row0, n, h, delta, y0, EPS, ws)
    assert torch.equal(y, y0)
    for a, b in zip(got, (h, k, v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    m = n if voters is None else min(voters, n)
    if m == 0:
        assert torch.equal(w, before)
        return
    added, rel = weights64(q[n - m:], k[:, :rows].double(), rows - m)
    check(w[:, :rows], before[:, :rows], added, rel)
    assert torch.equal(w[:, rows:], before[:, rows:])


@pytest.mark.parametrize("how", ["small scratch", "none"])
def test_layer_prefill_weights_without_voters(attn, layers, how):
    """The chunks of a prompt before the one that votes: what only votes need is not asked for."""
    g = gen(8)
    row0, n = 40, 20
    ctx = row0 + n + 2
    k, v = f16_cache(g, row0, ctx)
    h = randn(g, n * 2048)
    got = [t.clone() for t in (h, k, v)]
    ws = attn.LayerWorkspace(max_tok=32)
    y, y0 = (torch.empty(n * 2048, device="cuda") for _ in range(2))
    votes = (None, None) if how == "none" else \
        (torch.empty(0, device="cuda"), attn.PrefillWeightsScratch(4, 8))
    attn.layer_prefill_weights(layers["q4_k"], got[1], got[2], ctx, row0, row0, n, got[0], None, y, EPS,
                               ws, *votes, voters=0)
    attn.layer_prefill(layers["q4_k"], k, v, ctx, row0, n, h, None, y0, EPS, ws)
    assert torch.equal(y, y0)
    for a, b in zip(got, (h, k, v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("row0,pos0,n", [(0, 50, 20), (100, 5000, 33)])
def test_layer_prefill_weights_at_another_row(attn, layers, row0, pos0, n):
    g = gen(pos0)
    ctx, big = row0 + n + 3, pos0 + n
    k, v = f16_cache(g, row0, ctx)
    old = [k.clone(), v.clone()]
    kb, vb = f16_cache(g, pos0, big)
    h = randn(g, n * 2048)
    ws, sc = attn.LayerWorkspace(max_tok=64), attn.PrefillWeightsScratch(n, row0 + n)
    w, y = torch.zeros(KV, ctx, device="cuda"), torch.empty(n * 2048, device="cuda")
    attn.layer_prefill(layers["q4_k"], kb, vb, big, pos0, n, h.clone(), None, y, EPS, ws)
    q0 = prefill_queries(attn, ws, n)
    attn.layer_prefill_weights(layers["q4_k"], k, v, ctx, row0, pos0, n, h, None, y, EPS, ws, w, sc)
    assert torch.equal(q0, prefill_queries(attn, ws, n))  # rotated for the positions
    for a, b, c in ((k, kb, old[0]), (v, vb, old[1])):
        assert torch.equal(a[:, row0:row0 + n], b[:, pos0:pos0 + n])
        assert torch.equal(a[:, :row0], c[:, :row0])
        assert torch.equal(a[:, row0 + n:].view(torch.uint8), c[:, row0 + n:].view(torch.uint8))
    k64, v64 = (t[:, :row0 + n].double() for t in (k, v))
    added, rel = weights64(q0, k64, row0)
    check(w[:, :row0 + n], torch.zeros_like(w[:, :row0 + n]), added, rel)
    qg = ws.prefill[:n * 9216].view(n, 9216)[:, :8192].reshape(n, H, 2, D)
    want = attend64(q0, qg, k64, v64, row0)
    core = ws.prefill_core[:n].view(n, H, D).double()
    # the causal prefill's own gate (f16 queries and numerators)
    assert float((core - want).norm() / want.norm()) <= 5e-3


def test_layer_refusals(attn, layers):
    f32 = dict(dtype=torch.float32, device="cuda")
    k = torch.zeros(KV, 64, D, dtype=torch.float16, device="cuda")
    h, y, w = torch.zeros(4 * 2048, **f32), torch.zeros(4 * 2048, **f32), torch.zeros(KV, 64, **f32)
    ws = attn.LayerWorkspace(max_tok=16)
    sc, psc = attn.DecodeWeightsScratch(128, 32), attn.PrefillWeightsScratch(2, 32)
    args = (layers["q4_k"], k, k.clone(), 64)
    with pytest.raises(ValueError):  # beyond the scratch
        attn.layer_decode_weights(*args, 32, 32, h, None, y, EPS, ws, w, sc)
    with pytest.raises(ValueError):
        attn.layer_decode_weights(*args, 20, 20, h, None, y, EPS, ws, w,
                                  attn.DecodeWeightsScratch(0, 32))
    with pytest.raises(ValueError):
        attn.layer_prefill_weights(*args, 0, 0, 4, h, None, y, EPS, ws, w, psc)
    with pytest.raises(RuntimeError):  # the cache is full
        attn.layer_decode_weights(layers["q4_k"], k, k.clone(), 20, 20, 90, h, None, y, EPS, ws, w,
                                  sc)
    with pytest.raises(RuntimeError):  # a position behind its row
        attn.layer_prefill_weights(*args, 5, 4, 2, h, None, y, EPS, ws, w, psc)
    with pytest.raises(RuntimeError):
        attn.layer_prefill_weights(*args, 0, 0, 4, h, None, y, EPS, attn.LayerWorkspace(max_tok=2), w,
                                   attn.PrefillWeightsScratch(4, 32))
