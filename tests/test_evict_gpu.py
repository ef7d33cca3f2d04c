"""GPU tests of the bounded cache: accumulated attention weights (decode, prompt chunks), the rows
to keep, their move, the appends behind it, and all of them together, against float64.

Tolerance of a weight. A score in log2 units is a sum of 256 products q k log2(e) / 16 with
A = sum |q k| log2(e) / 16 the sum of their magnitudes. The query's f16 pair is off by at most 2^-22
of each product and the f32 sums (at most 40 of them after one another: the k-steps of the matrix
products, twice, and the exponent's fma) by 40 half steps of A; the exponential, the maximum's and the
sum's own share are as large again. A weight is therefore off by at most
  rel = 2 ln 2 A (2^-22 + 40 2^-24)
of itself, and its sum over queries by as many half steps of 2^-24 as it has terms after one another
(at most one per block of 4 tokens, and 64 in the joins).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

H, KV, G, D = 16, 2, 8, 256


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, dtype=dtype, device="cuda")


def weights64(q, k, pos0):
    """Sums [2][keys] of the causal weights of q [n][16][256] over k [2][keys][256] (float64; token
    t sees keys up to pos0 + t), and the tolerance of the module's docstring for them."""
    n, keys = q.shape[0], k.shape[1]
    out = torch.zeros(KV, keys, dtype=torch.float64, device="cuda")
    top = 0.0
    seen = pos0 + torch.arange(n, device="cuda")
    hidden = torch.arange(keys, device="cuda")[None, :] > seen[:, None]
    for h in range(H):
        s = (q[:, h].double() @ k[h // G].T) / math.sqrt(D)
        s.masked_fill_(hidden, -math.inf)
        out[h // G] += torch.softmax(s, dim=1).sum(dim=0)
        mag = (q[:, h].double().abs() @ k[h // G].abs().T).masked_fill_(hidden, 0.0)
        top = max(top, float(mag.max()) / math.sqrt(D) * math.log2(math.e))
    rel = 2 * math.log(2) * top * (2 ** -22 + 40 * 2 ** -24)
    return out, rel + (n / 4 + 64) * 2 ** -24


def check(got, before, added, rel, name=""):
    """got = before + added within rel of added and half a step of the sum."""
    want = before.double() + added
    off = (got.double() - want).abs()
    lim = rel * added + 2 ** -23 * want.abs() + 1e-30
    assert torch.isfinite(got).all(), name
    worst = float((off / lim).max())
    assert worst <= 1, (name, worst)


def e4m3_rows(g, rows):
    x = randn(g, KV, rows, D)
    scale = torch.exp2(torch.floor(torch.log2(x.abs().amax(dim=-1, keepdim=True))) - 7)
    codes = (x / scale).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), scale[..., 0].contiguous(), codes.float().double() * scale.double()


def fp8_cache(attn, g, rows, max_ctx):
    """A cache of max_ctx rows whose first `rows` are random, the others NaN codes and scales."""
    c = attn.Fp8Cache(max_ctx)
    k8, ks, k = e4m3_rows(g, rows)
    v8, vs, v = e4m3_rows(g, rows)
    for t, x in ((c.k8, k8), (c.v8, v8)):
        t.fill_(0x7F)
        t.view(KV, max_ctx, D)[:, :rows] = x
    for t, x in ((c.k_scale, ks), (c.v_scale, vs)):
        t.fill_(math.nan)
        t.view(KV, max_ctx)[:, :rows] = x
    return c, k, v


def f16_cache(g, rows, max_ctx):
    """K, V [2][max_ctx][256] f16, the rows past `rows` NaN."""
    out = []
    for _ in range(2):
        x = torch.full((KV, max_ctx, D), math.nan, dtype=torch.float16, device="cuda")
        x[:, :rows] = randn(g, KV, rows, D, dtype=torch.float16)
        out.append(x)
    return out


LENS = [1, 2, 7, 8, 31, 32, 33, 63, 255, 257, 1000, 4097, 33001]


@pytest.mark.parametrize("n", LENS)
def test_decode_weights(attn, n):
    g = gen(n)
    ctx = n + 13
    q, qg = 2.0 * randn(g, H, D), randn(g, H, 2, D)
    k, v = f16_cache(g, n, ctx)
    before = torch.rand(KV, ctx, generator=g, device="cuda") * (8.0 / n)
    sc = attn.DecodeWeightsScratch(200, ctx)
    added, rel = weights64(q[None], k[:, :n].double(), n - 1)
    core, core0 = torch.empty(H, D, device="cuda"), torch.empty(H, D, device="cuda")
    for n_splits in (None, 1, 3, 60, 200):
        w = before.clone()
        used = attn.attn_decode_weights(q, qg, k, v, core, w, sc, n, ctx, n_splits=n_splits)
        attn.attn_decode(q, qg, k, v, core0, sc, n, ctx, n_splits=used)
        assert torch.equal(core, core0)
        check(w[:, :n], before[:, :n], added, rel, (n, n_splits))
        assert torch.equal(w[:, n:], before[:, n:])
        again = before.clone()
        attn.attn_decode_weights(q, qg, k, v, core, again, sc, n, ctx, n_splits=n_splits)
        assert torch.equal(w, again)
        attn.attn_decode_weights(q, qg, k, v, core, again, sc, n, ctx, n_splits=n_splits)
        check(again[:, :n], w[:, :n], added, rel, "accumulated")


@pytest.mark.parametrize("n", LENS)
def test_decode_weights_fp8(attn, n):
    g = gen(100 + n)
    ctx = n + 5
    q, qg = 2.0 * randn(g, H, D), randn(g, H, 2, D)
    cache, k, _ = fp8_cache(attn, g, n, ctx)
    before = torch.rand(KV, ctx, generator=g, device="cuda") * (8.0 / n)
    sc = attn.DecodeWeightsScratch(128, ctx)
    added, rel = weights64(q[None], k, n - 1)
    core, core0 = torch.empty(H, D, device="cuda"), torch.empty(H, D, device="cuda")
    for n_splits in (None, 1, 5):
        w = before.clone()
        used = attn.attn_decode_weights_fp8(q, qg, cache, core, w, sc, n, n_splits=n_splits)
        attn.attn_decode_fp8(q, qg, cache, core0, sc, n, n_splits=used)
        assert torch.equal(core, core0)
        check(w[:, :n], before[:, :n], added, rel, (n, n_splits))
        assert torch.equal(w[:, n:], before[:, n:])


def test_decode_weights_peaked(attn):
    """One key takes nearly everything; rising and falling scores move the running maxima."""
    g = gen(5)
    n = 3001
    q, qg = 6.0 * randn(g, H, D), randn(g, H, 2, D)
    k, v = f16_cache(g, n, n)
    ramp = torch.linspace(0.1, 1.0, n, device="cuda")
    for order in (ramp, ramp.flip(0)):
        kk = (k.float() * order[None, :, None]).half()
        w = torch.zeros(KV, n, device="cuda")
        sc = attn.DecodeWeightsScratch(64, n)
        attn.attn_decode_weights(q, qg, kk, v, torch.empty(H, D, device="cuda"), w, sc, n, n)
        added, rel = weights64(q[None], kk.double(), n - 1)
        check(w, torch.zeros_like(w), added, rel)


CHUNKS = [(0, 1), (0, 2), (5, 1), (0, 4), (0, 5), (0, 33), (31, 2), (32, 1), (61, 7), (1000, 3),
          (100, 301), (12001, 33), (0, 1024), (77, 1500), (3000, 2049), (4100, 17), (5003, 300),
          (40000, 3)]


@pytest.mark.parametrize("pos0,n", CHUNKS)
@pytest.mark.parametrize("fp8", [False, True])
def test_prefill_weights(attn, pos0, n, fp8):
    g = gen(pos0 + 7 * n)
    rows, ctx = pos0 + n, pos0 + n + 11
    q = 2.0 * randn(g, n, H, D)
    before = torch.rand(KV, ctx, generator=g, device="cuda") * (8.0 * n / rows)
    sc = attn.PrefillWeightsScratch(n, rows, fp8=fp8)
    sc.ws.fill_(0xFF)  # a workspace of NaN
    if fp8:
        cache, k, _ = fp8_cache(attn, g, rows, ctx)
        call = lambda w: attn.attn_prefill_weights_fp8(q, cache, w, pos0, n, sc)  # noqa: E731
    else:
        kc, _ = f16_cache(g, rows, ctx)
        k = kc[:, :rows].double()
        call = lambda w: attn.attn_prefill_weights(q, kc, w, pos0, n, ctx, sc)  # noqa: E731
    added, rel = weights64(q, k, pos0)
    w, again = before.clone(), before.clone()
    call(w)
    call(again)
    check(w[:, :rows], before[:, :rows], added, rel, (pos0, n))
    assert torch.equal(w[:, rows:], before[:, rows:])
    assert torch.equal(w, again)


def test_prefill_weights_with_a_larger_scratch(attn):
    """The scratch of a large chunk serves every smaller one, whatever the chunk before left in it."""
    g = gen(9)
    sc = attn.PrefillWeightsScratch(700, 2000)
    for pos0, n in ((1300, 700), (0, 3), (900, 40), (1999, 1), (0, 700)):
        rows = pos0 + n
        kc, _ = f16_cache(g, rows, 2000)
        q = 2.0 * randn(g, n, H, D)
        w = torch.zeros(KV, 2000, device="cuda")
        attn.attn_prefill_weights(q, kc, w, pos0, n, 2000, sc)
        added, rel = weights64(q, kc[:, :rows].double(), pos0)
        check(w[:, :rows], torch.zeros_like(w[:, :rows]), added, rel, (pos0, n))


@pytest.mark.parametrize("fp8", [False, True])
def test_prefill_weights_in_pieces(attn, fp8):
    """A chunk over a cache so long that it runs in two pieces."""
    g = gen(10)
    pos0, n = 66000, 4000
    rows = pos0 + n
    q = 2.0 * randn(g, n, H, D)
    w = torch.zeros(KV, rows, device="cuda")
    sc = attn.PrefillWeightsScratch(n, rows, fp8=fp8)
    sc.ws.fill_(0xFF)  # a workspace of NaN
    if fp8:
        cache, k, _ = fp8_cache(attn, g, rows, rows)
        attn.attn_prefill_weights_fp8(q, cache, w, pos0, n, sc)
    else:
        k, _ = f16_cache(g, rows, rows)
        attn.attn_prefill_weights(q, k, w, pos0, n, rows, sc)
    added, rel = weights64(q, k.double(), pos0)
    check(w, torch.zeros_like(w), added, rel)


@pytest.mark.parametrize("rows,n", [(1_000_000, 130), (1_100_001, 300), (4_200_000, 16)])
def test_prefill_weights_over_a_million_rows(attn, rows, n):
    """Groups that the bound of their sums makes larger, pieces of 8 groups with a rest, one group."""
    g = gen(rows)
    k = randn(g, KV, rows, D, dtype=torch.float16)
    q = 2.0 * randn(g, n, H, D)
    w = torch.zeros(KV, rows, device="cuda")
    sc = attn.PrefillWeightsScratch(n, rows)
    sc.ws.fill_(0xFF)  # a workspace of NaN
    attn.attn_prefill_weights(q, k, w, rows - n, n, rows, sc)
    added, rel = weights64(q, k.double(), rows - n)
    check(w, torch.zeros_like(w), added, rel)


@pytest.mark.parametrize("pos0,n", [(2500, 70), (5000, 300), (0, 200)])
def test_prefill_weights_peaked(attn, pos0, n):
    """Few keys take nearly everything; rising scores lead the first tile's by far more and by less
    than 2^40, falling ones leave the later tiles next to nothing."""
    g = gen(pos0 + 13)
    rows = pos0 + n
    kc, _ = f16_cache(g, rows, rows)
    q = randn(g, n, H, D)
    q[::2] *= 6.0
    ramp = torch.linspace(0.1, 1.0, rows, device="cuda")
    for order in (ramp, ramp.flip(0)):
        kk = (kc.float() * order[None, :, None]).half()
        w = torch.zeros(KV, rows, device="cuda")
        attn.attn_prefill_weights(q, kk, w, pos0, n, rows, attn.PrefillWeightsScratch(n, rows))
        added, rel = weights64(q, kk.double(), pos0)
        check(w, torch.zeros_like(w), added, rel)


def test_prefill_weights_query_magnitudes(attn):
    """Rows of zeros (every key alike), rows far apart in magnitude, and elements far below their
    row's largest."""
    g = gen(11)
    pos0, n = 200, 40
    rows = pos0 + n
    kc, _ = f16_cache(g, rows, rows)
    q = randn(g, n, H, D)
    q[0] = 0.0
    q[1] *= 1e-30
    q[2] *= 30.0
    q[3, :, 1:] *= 1e-6
    q[4] *= 2.0 ** -100
    q[5, :8] = 0.0
    w = torch.zeros(KV, rows, device="cuda")
    attn.attn_prefill_weights(q, kc, w, pos0, n, rows, attn.PrefillWeightsScratch(n, rows))
    added, rel = weights64(q, kc.double(), pos0)
    check(w, torch.zeros_like(w), added, rel)


def limit64(q, k, pos0, k_off=0.0):
    """weights64's sums, and how far each may be off, query by query: a score in log2 units by
      A (2^-22 + 40 2^-24) + (2^-38 B sum |k| + k_off sum |q|) log2(e) / 16
    (A the sum of the magnitudes of its products as in the module's docstring; B the largest query element
    of its block of 4 tokens x 8 heads, whose power of two the cut shares; k_off what a K element is off
    by), its logarithmic sum by the largest of these, its weight by 2^(both) - 1 of itself, and by 2^-19
    of itself for the exponential, the sums of the statistics and the scale's rounding."""
    n, keys = q.shape[0], k.shape[1]
    out = torch.zeros(KV, keys, dtype=torch.float64, device="cuda")
    lim = torch.zeros_like(out)
    hidden = torch.arange(keys, device="cuda")[None, :] > \
        pos0 + torch.arange(n, device="cuda")[:, None]
    top = q.abs().amax(dim=2).view(n, KV, G).amax(dim=2)
    for h in range(H):
        kk = k[h // G]
        s = (q[:, h].double() @ kk.T) / math.sqrt(D)
        p = torch.softmax(s.masked_fill_(hidden, -math.inf), dim=1)
        out[h // G] += p.sum(dim=0)
        block = torch.stack([top[t // 4 * 4:t // 4 * 4 + 4, h // G].max() for t in range(n)]).double()
        off = (q[:, h].double().abs() @ kk.abs().T) * (2 ** -22 + 40 * 2 ** -24)
        off += 2 ** -38 * block[:, None] * kk.abs().sum(dim=1)
        off += k_off * q[:, h].double().abs().sum(dim=1)[:, None]
        off = (off * (math.log2(math.e) / math.sqrt(D))).masked_fill_(hidden, 0.0)
        off += off.amax(dim=1, keepdim=True)
        lim[h // G] += (p * torch.expm1(off * math.log(2) + 2 ** -19)).clamp(max=1.0).sum(dim=0)
    return out, lim + (n / 4 + 64) * 2 ** -24 * out + 1e-30


@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 16, 2.0 ** 22])
@pytest.mark.parametrize("t,h", [(0, 0), (5, 3), (6, 12)])
def test_prefill_weights_of_one_large_query(attn, factor, t, h):
    """One head of one token far larger than the others: what it takes from the precision of its block's
    queries is bounded, and those of other blocks keep theirs (limit64)."""
    g = gen(t + h)
    pos0, n = 190, 12
    rows = pos0 + n
    kc, _ = f16_cache(g, rows, rows)
    q = randn(g, n, H, D)
    q[t, h] *= factor
    w = torch.zeros(KV, rows, device="cuda")
    attn.attn_prefill_weights(q, kc, w, pos0, n, rows, attn.PrefillWeightsScratch(n, rows))
    want, lim = limit64(q, kc.double(), pos0)
    assert float(((w.double() - want).abs() / lim).max()) <= 1


def one_row_takes_all(g, pos0, n, size):
    """Queries so large that each gives all its weight to one row: rows k = (a | b) s with s a vector of
    signs and the levels a + b distinct whole numbers, queries +-size s. Scores are 8 size (a + b): they
    lie 8 size apart, and at most 3000 times that from 0, so that f32 tells them apart. Returns q, K and
    the weights, whole numbers."""
    rows = pos0 + n
    level = torch.stack([torch.randperm(6000, generator=g, device="cuda")[:rows] for _ in range(KV)])
    a, b = level % 2000 - 1000, level // 2000 * 2000 - 2000
    sign = torch.where(torch.rand(D, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    k = torch.stack([a, b], dim=2).repeat_interleave(D // 2, dim=2).float() * sign
    way = torch.where(torch.rand(n, H, generator=g, device="cuda") < 0.5, -1, 1)
    want = torch.zeros(KV, rows, device="cuda")
    for t in range(n):
        for h in range(H):
            seen = (way[t, h] * (a + b)[h // G])[:pos0 + t + 1]
            want[h // G, seen.argmax()] += 1
    return size * way[..., None] * sign, k.half(), want


SIZES = [2.0 ** 4, 2.0 ** 12, 2.0 ** 25, 2.0 ** 40, 2.0 ** 70, 2.0 ** 110]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("pos0,n", [(300, 33), (0, 70), (5000, 9)])
def test_prefill_weights_of_large_queries(attn, pos0, n, size):
    """Scores up to 2^124: the largest one's weight is 1, the others' 0, no infinity and no NaN."""
    q, k, want = one_row_takes_all(gen(n), pos0, n, size)
    w = torch.zeros_like(want)
    attn.attn_prefill_weights(q, k, w, pos0, n, pos0 + n, attn.PrefillWeightsScratch(n, pos0 + n))
    assert torch.equal(w, want), (float(w.max()), float((w - want).abs().max()))


@pytest.mark.parametrize("size", [2.0 ** 4, 2.0 ** 12, 2.0 ** 18])
@pytest.mark.parametrize("n", [1, 70, 5009])
def test_decode_weights_of_large_queries(attn, n, size):
    """The decodes take queries below 2^19."""
    q, k, want = one_row_takes_all(gen(n), n - 1, 1, size)
    w = torch.zeros_like(want)
    core, qg = torch.empty(H, D, device="cuda"), torch.zeros(H, 2, D, device="cuda")
    attn.attn_decode_weights(q[0], qg, k, k, core, w, attn.DecodeWeightsScratch(64, n), n, n)
    assert torch.equal(w, want), (float(w.max()), float((w - want).abs().max()))


@pytest.mark.parametrize("pos0,n", [(0, 300), (700, 33), (4000, 300), (2000, 4)])
def test_prefill_weights_of_low_halves(attn, pos0, n):
    """Queries whose elements need more than f16: all of (1 + 2^-12) times a power of two. Without the
    second half every score of a token would be 2^-12 of itself nearer to 0, for all tokens alike, and
    weights off by up to 2^-12 times 32 of themselves, 46 times the tolerance."""
    g = gen(n)
    rows = pos0 + n
    level = torch.rand(KV, rows, 1, generator=g, device="cuda") * 2 - 1
    sign = torch.where(torch.rand(D, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    kc = (level * sign).half()
    q = torch.exp2(torch.randint(-1, 2, (n, H, 1), generator=g, device="cuda").float())
    q = q * (1 + 2 ** -12) * sign
    w = torch.zeros(KV, rows, device="cuda")
    attn.attn_prefill_weights(q, kc, w, pos0, n, rows, attn.PrefillWeightsScratch(n, rows))
    added, rel = weights64(q, kc.double(), pos0)
    check(w, torch.zeros_like(w), added, rel)


@pytest.mark.parametrize("low,high,size", [(-30, -9, 50.0), (5, 11, 2.0 ** -13),
                                           (12, 17, 2.0 ** -15)])
@pytest.mark.parametrize("pos0,n", [(300, 40), (0, 33)])
def test_prefill_weights_fp8_row_scales(attn, low, high, size, pos0, n):
    """Rows of very small and very large scales: K as f16, its elements off by at most 2^-25 where f16 is
    subnormal (4 bits of a code are exact elsewhere) and held within 65504."""
    g = gen(low + n)
    rows = pos0 + n
    cache, k, _ = fp8_cache(attn, g, rows, rows)
    more = torch.exp2(torch.randint(low, high, (KV, rows), generator=g, device="cuda").float())
    cache.k_scale.mul_(more.view(-1))
    k = k * more.double()[..., None]
    assert (low == 12) == (float(k.abs().max()) > 65504)
    q = size * randn(g, n, H, D)
    w = torch.zeros(KV, rows, device="cuda")
    attn.attn_prefill_weights_fp8(q, cache, w, pos0, n,
                                  attn.PrefillWeightsScratch(n, rows, fp8=True))
    want, lim = limit64(q, k.clamp(-65504.0, 65504.0), pos0, 2 ** -25)
    assert float(((w.double() - want).abs() / lim).max()) <= 1


def test_prefill_weights_of_one_token_equals_decode(attn):
    g = gen(12)
    n = 777
    q, qg = 2.0 * randn(g, 1, H, D), randn(g, H, 2, D)
    k, v = f16_cache(g, n, n)
    a, b = torch.zeros(KV, n, device="cuda"), torch.zeros(KV, n, device="cuda")
    attn.attn_prefill_weights(q, k, a, n - 1, 1, n, attn.PrefillWeightsScratch(1, n))
    attn.attn_decode_weights(q, qg, k, v, torch.empty(H, D, device="cuda"), b,
                             attn.DecodeWeightsScratch(64, n), n, n)
    added, rel = weights64(q, k.double(), n - 1)
    zero = torch.zeros_like(a)
    check(a, zero, added, rel)
    check(b, zero, added, rel)


def select_np(w, keep, sinks, recent):
    """Kept rows of one head: by (weight descending, NaN last, row)."""
    n = len(w)
    rank = np.where(np.isnan(w), -np.inf, w.astype(np.float64))
    tier = np.where(np.isnan(w), 0, 1)  # a NaN ranks below -inf
    tier[:sinks] = 2
    tier[n - recent:] = 2
    order = np.lexsort((np.arange(n), -rank, -tier))
    return np.sort(order[:keep])


def run_select(attn, w, n, keep, sinks, recent, max_len=None):
    ctx = w.shape[1]
    index = torch.full((KV * keep + 3,), -7, dtype=torch.int32, device="cuda")
    attn.attn_evict_select(w, n, ctx, keep, sinks, recent, index, attn.EvictScratch(max_len or n))
    assert (index[KV * keep:] == -7).all()
    return index[:KV * keep].view(KV, keep).cpu().numpy()


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 1000, 1023, 1024, 1025, 2048, 2049, 5000, 8192,
                               8193, 16384, 16385, 16411, 17409, 32768, 40001, 65536, 65537, 131071,
                               262144])
def test_select(attn, n):
    rng = np.random.default_rng(n)
    ctx = n + 3
    w = np.exp(2 * rng.standard_normal((KV, ctx))).astype(np.float32)
    w[:, rng.random(ctx) < 0.1] = 0.0
    w[:, n:] = 1e30  # rows past the sequence are not looked at
    wd = torch.from_numpy(w).cuda()
    for keep in sorted({1, (n + 1) // 2, max(1, n // 10), max(1, n - 1), n}):
        for sinks, recent in ((0, 0), (min(4, keep), 0), (0, keep), (keep, 0),
                              (min(4, keep), min(100, keep - min(4, keep)))):
            got = run_select(attn, wd, n, keep, sinks, recent)
            for h in range(KV):
                assert np.array_equal(got[h], select_np(w[h, :n], keep, sinks, recent)), \
                    (n, keep, sinks, recent, h)


@pytest.mark.parametrize("n", [10, 1000, 20000, 100000])
def test_select_ties_and_specials(attn, n):
    rng = np.random.default_rng(n + 1)
    few = rng.choice(np.float32([0.0, -0.0, 1.0, 2.0]), (KV, n))
    odd = rng.choice(np.float32([0.0, -0.0, -1.0, 1e-42, -1e-42, 3.0, np.inf, -np.inf, np.nan]), (KV, n))
    same = np.full((KV, n), 0.25, np.float32)
    nans = np.full((KV, n), np.nan, np.float32)
    nans[0] = -np.float32(np.nan)
    for w in (few, odd, same, nans):
        for keep, sinks, recent in ((n // 2, 0, 0), (n // 3 + 1, 2, 1), (n - 1, 1, 3)):
            got = run_select(attn, torch.from_numpy(w).cuda(), n, keep, sinks, recent, 2 * n)
            for h in range(KV):
                assert np.array_equal(got[h], select_np(w[h], keep, sinks, recent)), (n, keep, h)


def test_select_of_long_stretches(attn):
    """Workgroups of more rows than a wave loads at a time."""
    n = 1500001
    rng = np.random.default_rng(4)
    spread = np.exp(2 * rng.standard_normal((KV, n))).astype(np.float32)
    close = (1.0 + 1e-5 * rng.random((KV, n))).astype(np.float32)  # many equal, one digit apart
    for w, keep, sinks, recent in ((spread, 700001, 4, 100), (close, 1000, 0, 0),
                                   (close, n - 5, 1, 2)):
        got = run_select(attn, torch.from_numpy(w).cuda(), n, keep, sinks, recent)
        for h in range(KV):
            assert np.array_equal(got[h], select_np(w[h], keep, sinks, recent)), (keep, h)


def test_select_lengths_of_one_scratch(attn):
    """One scratch, dirty at first, for selections of other numbers of workgroups in turn, of one launch
    and of four, eager and replayed: where a workspace's parts lie goes with the length."""
    rng = np.random.default_rng(6)
    ctx, esc = 90000, attn.EvictScratch(90000)
    esc.ws.fill_(0xFF)
    w = np.exp(rng.standard_normal((KV, ctx))).astype(np.float32)
    wd = torch.from_numpy(w).cuda()
    calls = []
    for n, keep in ((90000, 40001), (17000, 16999), (40000, 100), (16000, 9), (65537, 65000), (17408, 1)):
        index = torch.full((KV, keep), -7, dtype=torch.int32, device="cuda")
        want = np.stack([select_np(w[h, :n], keep, 3, 0 if keep < 10 else 5)
                         if keep > 3 else select_np(w[h, :n], keep, 0, 0) for h in range(KV)])
        args = (n, ctx, keep, 3 if keep > 3 else 0, 5 if keep >= 10 else 0, index)
        calls.append((args, index, want))
    graphs = []
    for args, index, want in calls:
        attn.attn_evict_select(wd, *args, esc)
        assert np.array_equal(index.cpu().numpy(), want), args[:3]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn.attn_evict_select(wd, *args, esc)
        graphs.append(graph)
    for order in (range(6), (5, 0, 1, 4, 2, 3)):
        for i in order:
            calls[i][1].fill_(-7)
            graphs[i].replay()
        for args, index, want in calls:
            assert np.array_equal(index.cpu().numpy(), want), args[:3]


GATHERS = [(1, 1, 1), (5, 3, 3), (64, 64, 70), (1000, 257, 300), (4099, 1023, 5000),
           (33000, 16001, 16384)]


@pytest.mark.parametrize("n,keep,out_ctx", GATHERS)
def test_gather(attn, n, keep, out_ctx):
    g = gen(n + keep)
    k, v = f16_cache(g, n, n)
    w = torch.rand(KV, n, generator=g, device="cuda")
    index = torch.stack([torch.randperm(n, generator=g, device="cuda")[:keep] for _ in range(KV)])
    index = index.to(torch.int32).contiguous()
    if keep > 2:
        index[0, 1] = -1  # not a row
        index[1, 2] = n
        index[1, 0] = index[1, 1]  # the same row twice
    ko, vo = (torch.full((KV, out_ctx, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    wo = torch.full((KV, out_ctx), 9.0, device="cuda")
    attn.attn_evict_gather(k, v, w, n, index, keep, ko, vo, wo, out_ctx)
    good = (index >= 0) & (index < n)
    at = torch.where(good, index, 0).long()
    head = torch.arange(KV, device="cuda")[:, None]
    for src, dst in ((k, ko), (v, vo)):
        want = torch.where(good[..., None], src[head, at], torch.zeros_like(src[head, at]))
        assert torch.equal(dst[:, :keep], want)
        assert (dst[:, keep:] == 3.0).all()
    assert torch.equal(wo[:, :keep], torch.where(good, w[head, at], torch.zeros_like(w[head, at])))
    assert (wo[:, keep:] == 0).all()


@pytest.mark.parametrize("n,keep,out_ctx", GATHERS)
def test_gather_fp8(attn, n, keep, out_ctx):
    g = gen(n + keep + 1)
    src, dst = attn.Fp8Cache(n), attn.Fp8Cache(out_ctx)
    for t in src.buffers():
        t.copy_(torch.randint(0, 250, t.shape, generator=g, device="cuda"))
    for t in dst.buffers():
        t.fill_(3)
    w = torch.rand(KV, n, generator=g, device="cuda")
    wo = torch.full((KV, out_ctx), 9.0, device="cuda")
    index = torch.stack([torch.randperm(n, generator=g, device="cuda")[:keep] for _ in range(KV)])
    index = index.to(torch.int32).contiguous()
    if keep > 2:
        index[0, 0] = 0x7FFFFFFF
    attn.attn_evict_gather_fp8(src, w, index, keep, dst, wo)
    good = (index >= 0) & (index < n)
    at = torch.where(good, index, 0).long()
    head = torch.arange(KV, device="cuda")[:, None]
    for a, b in zip((*src.buffers(), w), (*dst.buffers(), wo)):
        a, b = a.view(KV, n, -1), b.view(KV, out_ctx, -1)
        want = torch.where(good[..., None], a[head, at], torch.zeros_like(a[head, at]))
        assert torch.equal(b[:, :keep], want)
        assert (b[:, keep:] == (0 if a.data_ptr() == w.data_ptr() else 3)).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("keep,out_ctx", [(3, 20000), (1, 1025), (16, 262144), (500, 300001)])
def test_small_move_into_a_large_cache(attn, keep, out_ctx, fp8):
    """The weights behind the kept rows become 0, all of them and nothing else, and their clearing
    does not set the pace (it is 2 MB for 262144 rows): a move into a cache of that size takes at most
    4 times what the same move takes into one of its own size, by the least of several timings."""
    g = gen(keep + out_ctx)
    n = 600
    w = torch.rand(KV, n, generator=g, device="cuda")
    index = torch.stack([torch.randperm(n, generator=g, device="cuda")[:keep] for _ in range(KV)])
    index = index.to(torch.int32).contiguous()
    src = fp8_cache(attn, g, n, n)[0] if fp8 else f16_cache(g, n, n)

    def into(rows):
        guarded = torch.full((KV * rows + 64,), 9.0, device="cuda")
        wo = guarded[32:32 + KV * rows]
        if fp8:
            out = attn.Fp8Cache(rows)
            bufs = [t.fill_(3) for t in out.buffers()]
            return lambda: attn.attn_evict_gather_fp8(src, w, index, keep, out, wo), guarded, bufs
        bufs = [torch.full((KV, rows, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2)]
        return (lambda: attn.attn_evict_gather(*src, w, n, index, keep, *bufs, wo, rows)), guarded, bufs

    call, guarded, bufs = into(out_ctx)
    call()
    assert (guarded[:32] == 9).all() and (guarded[-32:] == 9).all()
    got = guarded[32:-32].view(KV, out_ctx)
    assert torch.equal(got[:, :keep], w[torch.arange(KV, device="cuda")[:, None], index.long()])
    assert (got[:, keep:] == 0).all()
    for t in bufs:
        assert (t.view(KV, out_ctx, -1)[:, keep:] == 3).all()

    def least(f):
        best = math.inf
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(20):
                f()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    small = into(keep)[0]
    least(small), least(call)  # both warm
    assert least(call) <= 4 * least(small)


@pytest.mark.parametrize("keep,hidden", [(33, range(33)), (70, range(40)), (200, range(64, 170)),
                                         (700, [*range(96), *range(300, 500), 699])])
def test_decode_over_gathered_rows_of_zeros(attn, keep, hidden):
    """Rows that an index outside the source left as zeros (e4m3: scale 0) are keys like others: score
    0, value 0. Whole tiles of them, also the first ones of a wave."""
    g = gen(keep)
    n = 900
    src, dst = fp8_cache(attn, g, n, n)[0], attn.Fp8Cache(keep)
    index = torch.stack([torch.randperm(n, generator=g, device="cuda")[:keep] for _ in range(KV)])
    index = index.to(torch.int32).contiguous()
    index[:, list(hidden)] = n
    attn.attn_evict_gather_fp8(src, torch.rand(KV, n, generator=g, device="cuda"), index, keep, dst,
                               torch.empty(KV, keep, device="cuda"))
    k, v = ((x.view(torch.float8_e4m3fn).float().double().view(KV, keep, D) *
             s.double().view(KV, keep, 1))
            for x, s in ((dst.k8, dst.k_scale), (dst.v8, dst.v_scale)))
    for t in (k, v):
        assert (t[:, list(hidden)] == 0).all()
    q, qg = 2.0 * randn(g, 1, H, D), randn(g, 1, H, 2, D)
    sc, zero = attn.DecodeWeightsScratch(8, keep), torch.zeros(KV, keep, device="cuda")
    added, rel = weights64(q, k, keep - 1)
    want = attend64(q, qg, k, v, keep - 1)[0]
    for n_splits in (1, 2, None):
        core, w = torch.empty(H, D, device="cuda"), zero.clone()
        attn.attn_decode_weights_fp8(q, qg, dst, core, w, sc, keep, n_splits=n_splits)
        check(w, zero, added, rel, n_splits)
        for h in range(H):  # the reference's gate for a decode
            err, size = (core[h].double() - want[h]).norm(), want[h].norm()
            assert float(err) <= 1e-5 * float(size), (n_splits, h)


def prep_inputs(g, n):
    proj = randn(g, n, 9216)
    norms = [1 + 0.1 * randn(g, D), 1 + 0.1 * randn(g, D)]
    i = torch.arange(32, dtype=torch.float64)
    return proj, norms, (1e7 ** (-i / 32)).float().cuda()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("pos,row", [(0, 0), (40, 40), (1000, 3), (5, 30), (100000, 0), (7, 43)])
def test_prep_at_another_row(attn, pos, row, fp8):
    """The row is the one that the prep writes at `pos`, bit for bit; no other row is touched."""
    g = gen(pos + row)
    ctx, m = 48, 4
    proj, norms, inv = prep_inputs(g, m)
    big = pos + m
    qg, k, v = proj[:, :8192], proj[:, 8192:8704], proj[:, 8704:9216]

    def one(t):
        return proj[t, :8192], proj[t, 8192:8704], proj[t, 8704:9216]

    def caches(rows):
        if fp8:
            c = attn.Fp8Cache(rows)
            for t in c.buffers():
                t.fill_(7)
            return c
        return [torch.full((KV, rows, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]

    def views(c, rows):
        return [t.view(KV, rows, -1) for t in (c.buffers() if fp8 else c)]

    far, near, single = caches(big), caches(ctx), caches(ctx)
    q0, q1, q2 = (torch.empty(m, H, D, device="cuda") for _ in range(3))
    if fp8:
        attn.attn_prep_batch_fp8(qg, k, v, *norms, inv, far, q0, pos, m, 9216)
        attn.attn_prep_batch_fp8(qg, k, v, *norms, inv, near, q1, pos, m, 9216, row0=row)
        for t in range(m):
            attn.attn_prep_fp8(*one(t), *norms, inv, single, q2[t], pos + t, row=row + t)
    else:
        attn.attn_prep_batch(qg, k, v, *norms, inv, *far, q0, pos, big, 1e-6, m, 9216)
        attn.attn_prep_batch(qg, k, v, *norms, inv, *near, q1, pos, ctx, 1e-6, m, 9216, row0=row)
        for t in range(m):
            attn.attn_prep(*one(t), *norms, inv, *single, q2[t], pos + t, ctx, 1e-6, row=row + t)
    assert torch.equal(q0, q1)
    assert torch.equal(q0, q2)
    for a, b, c in zip(views(far, big), views(near, ctx), views(single, ctx)):
        assert torch.equal(a[:, pos:pos + m], b[:, row:row + m])
        assert torch.equal(b, c)
        assert (b[:, :row] == 7).all() and (b[:, row + m:] == 7).all()


def attend64(q, qg, k, v, pos0):
    """Gated causal attention in float64: q [n][16][256], gate the second half of qg, k / v
    [2][keys][256]."""
    n, keys = q.shape[0], k.shape[1]
    hidden = torch.arange(keys, device="cuda")[None, :] > pos0 + torch.arange(n, device="cuda")[:, None]
    out = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
    for h in range(H):
        s = (q[:, h].double() @ k[h // G].T) / math.sqrt(D)
        out[:, h] = torch.softmax(s.masked_fill_(hidden, -math.inf), dim=1) @ v[h // G]
    return out * torch.sigmoid(qg[:, :, 1].double())


@pytest.mark.parametrize("fp8", [False, True])
def test_bounded_generation(attn, fp8):
    """A prompt, its votes, some tokens, an eviction into a smaller cache, more tokens and another
    eviction: each step against float64 over the rows that are then cached."""
    g = gen(77)
    prompt, ctx, small, keep = 300, 340, 128, 96
    proj, norms, inv = prep_inputs(g, 400)
    w = torch.zeros(KV, ctx, device="cuda")
    sc = attn.DecodeWeightsScratch(128, ctx)
    psc = attn.PrefillWeightsScratch(prompt, ctx, fp8=fp8)
    esc = attn.EvictScratch(ctx)
    index = torch.empty(KV, keep, dtype=torch.int32, device="cuda")
    make = (lambda n: attn.Fp8Cache(n)) if fp8 else \
        (lambda n: [torch.zeros(KV, n, D, dtype=torch.float16, device="cuda") for _ in range(2)])

    def values(c, n, rows):  # K, V in float64
        if fp8:
            return [(x.view(torch.float8_e4m3fn).float().double().view(KV, n, D) *
                     s.double().view(KV, n, 1))[:, :rows]
                    for x, s in ((c.k8, c.k_scale), (c.v8, c.v_scale))]
        return [x[:, :rows].double() for x in c]

    cache = make(ctx)
    q = torch.empty(prompt, H, D, device="cuda")
    args = (proj[:prompt, :8192], proj[:prompt, 8192:8704], proj[:prompt, 8704:], *norms, inv)
    if fp8:
        attn.attn_prep_batch_fp8(*args, cache, q, 0, prompt, 9216)
        attn.attn_prefill_weights_fp8(q, cache, w, 0, prompt, psc)
    else:
        attn.attn_prep_batch(*args, *cache, q, 0, ctx, 1e-6, prompt, 9216)
        attn.attn_prefill_weights(q, cache[0], w, 0, prompt, ctx, psc)
    k64, v64 = values(cache, ctx, prompt)
    added, rel = weights64(q, k64, 0)
    check(w[:, :prompt], torch.zeros_like(w[:, :prompt]), added, rel, "prompt")
    assert abs(float(w.double().sum()) - H * prompt) <= rel * H * prompt

    pos, rows, size = prompt, prompt, ctx
    q1, core = torch.empty(1, H, D, device="cuda"), torch.empty(1, H, D, device="cuda")
    for step in range(90):
        if rows == size - 1 or step == 20:  # full, or the first eviction, into the smaller cache
            kept = w.clone()
            attn.attn_evict_select(w, rows, size, keep, 4, 16, index, esc)
            want = [select_np(kept[h, :rows].cpu().numpy(), keep, 4, 16) for h in range(KV)]
            assert np.array_equal(index.cpu().numpy(), np.stack(want))
            out, w2 = make(small), torch.full((KV, small), 5.0, device="cuda")
            before = values(cache, size, rows)
            if fp8:
                attn.attn_evict_gather_fp8(cache, w, index, keep, out, w2)
            else:
                attn.attn_evict_gather(*cache, w, size, index, keep, *out, w2, small)
            cache, w, size, rows = out, w2, small, keep
            after = values(cache, size, keep)
            for a, b in zip(before, after):
                assert torch.equal(a[torch.arange(KV)[:, None], index.long()], b)
            assert (w[:, keep:] == 0).all()
        one = (proj[pos, :8192], proj[pos, 8192:8704], proj[pos, 8704:], *norms, inv)
        qg = proj[pos, :8192].contiguous()
        was = w.clone()
        if fp8:
            attn.attn_prep_fp8(*one, cache, q1, pos, row=rows)
            attn.attn_decode_weights_fp8(q1, qg, cache, core, w, sc, rows + 1)
        else:
            attn.attn_prep(*one, *cache, q1, pos, size, 1e-6, row=rows)
            attn.attn_decode_weights(q1, qg, *cache, core, w, sc, rows + 1, size)
        rows, pos = rows + 1, pos + 1
        k64, v64 = values(cache, size, rows)
        added, rel = weights64(q1, k64, rows - 1)
        check(w[:, :rows], was[:, :rows], added, rel, step)
        assert torch.equal(w[:, rows:], was[:, rows:])
        want = attend64(q1, qg.view(1, H, 2, D), k64, v64, rows - 1)
        for h in range(H):  # the reference's gate for a decode
            err = (core[0, h].double() - want[0, h]).norm() / want[0, h].norm()
            assert float(err) <= 1e-5


@pytest.mark.parametrize("n", [2500, 20001])  # a selection of one launch, of four
def test_captured_and_replayed(attn, n):
    """The operators in a graph on a stream of their own, replayed with other inputs between."""
    g = gen(31)
    m, keep = 40, 700
    q, qg = 2.0 * randn(g, m, H, D), randn(g, H, 2, D)
    k, v = f16_cache(g, n, n)
    w, core = torch.zeros(KV, n, device="cuda"), torch.empty(H, D, device="cuda")
    index = torch.zeros(KV, keep, dtype=torch.int32, device="cuda")
    ko, vo = (torch.zeros(KV, keep, D, dtype=torch.float16, device="cuda") for _ in range(2))
    wo = torch.zeros(KV, keep, device="cuda")
    sc, psc = attn.DecodeWeightsScratch(128, n), attn.PrefillWeightsScratch(m, n)
    esc = attn.EvictScratch(n)

    def step():
        attn.attn_prefill_weights(q, k, w, n - m, m, n, psc)
        attn.attn_decode_weights(q, qg, k, v, core, w, sc, n, n)
        attn.attn_evict_select(w, n, n, keep, 4, 64, index, esc)
        attn.attn_evict_gather(k, v, w, n, index, keep, ko, vo, wo, keep)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (1, 2, 3):
        h = gen(seed)
        q.copy_(2.0 * randn(h, m, H, D))
        k.copy_(randn(h, KV, n, D, dtype=torch.float16))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (core, w, index, ko, vo, wo)]
        w.zero_()
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (core, w, index, ko, vo, wo)):
            assert torch.equal(a, b)


def test_two_graphs_of_one_scratch(attn):
    """Two graphs captured over the same scratches, replayed in turn with eager calls between."""
    g = gen(32)
    n = 9000
    k, v = f16_cache(g, n, n)
    q, qg = 2.0 * randn(g, 70, H, D), randn(g, H, 2, D)
    sc, psc, esc = (attn.DecodeWeightsScratch(128, n), attn.PrefillWeightsScratch(70, n),
                    attn.EvictScratch(40000))

    def make(length, voters, keep):
        w, core = torch.zeros(KV, n, device="cuda"), torch.empty(H, D, device="cuda")
        index = torch.zeros(KV, keep, dtype=torch.int32, device="cuda")

        def step():
            attn.attn_prefill_weights(q, k, w, length - voters, voters, n, psc)
            attn.attn_decode_weights(q, qg, k, v, core, w, sc, length, n)
            attn.attn_evict_select(w, length, n, keep, 1, 8, index, esc)
        return step, (w, core, index)

    both = [make(n, 70, 4000), make(701, 3, 64)]
    graphs = []
    for step, _ in both:
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    for _ in range(3):
        for (step, out), graph in zip(both, graphs):
            out[0].zero_()
            graph.replay()
            got = [t.clone() for t in out]
            out[0].zero_()
            step()
            torch.cuda.synchronize()
            for a, b in zip(got, out):
                assert torch.equal(a, b)


def test_weights_and_indexes_need_no_alignment(attn):
    """Weights and indexes one element past an aligned address: the results of aligned ones."""
    g = gen(33)
    n, keep = 5001, 1203
    k, v = f16_cache(g, n, n)
    q, qg = 2.0 * randn(g, 20, H, D), randn(g, H, 2, D)
    core = torch.empty(H, D, device="cuda")
    sc, psc, esc = (attn.DecodeWeightsScratch(128, n), attn.PrefillWeightsScratch(20, n),
                    attn.EvictScratch(n))
    ko, vo = (torch.zeros(KV, keep, D, dtype=torch.float16, device="cuda") for _ in range(2))

    def run(off):
        w = torch.zeros(KV * n + 8, device="cuda")[off:off + KV * n]
        wo = torch.zeros(KV * keep + 8, device="cuda")[off:off + KV * keep]
        index = torch.zeros(KV * keep + 8, dtype=torch.int32, device="cuda")[off:off + KV * keep]
        attn.attn_prefill_weights(q, k, w, n - 20, 20, n, psc)
        attn.attn_decode_weights(q, qg, k, v, core, w, sc, n, n)
        attn.attn_evict_select(w, n, n, keep, 4, 100, index, esc)
        attn.attn_evict_gather(k, v, w, n, index, keep, ko, vo, wo, keep)
        return [t.clone() for t in (w, wo, index, ko, vo)]

    for a, b in zip(run(0), run(1)):
        assert torch.equal(a, b)


def test_two_streams_with_scratches_of_their_own(attn):
    g = gen(41)
    n = 20000
    q, qg = [2.0 * randn(g, 64, H, D) for _ in range(2)], randn(g, H, 2, D)
    k, v = f16_cache(g, n, n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def run(i, w, sc, psc, esc, index, core, stream):
        for _ in range(3):
            attn.attn_prefill_weights(q[i], k, w, n - 64, 64, n, psc, stream=stream)
            attn.attn_decode_weights(q[i], qg, k, v, core, w, sc, n, n, stream=stream)
            attn.attn_evict_select(w, n, n, n // 3, 4, 64, index, esc, stream=stream)

    def buffers():
        return (torch.zeros(KV, n, device="cuda"), attn.DecodeWeightsScratch(128, n),
                attn.PrefillWeightsScratch(64, n), attn.EvictScratch(n),
                torch.zeros(KV, n // 3, dtype=torch.int32, device="cuda"),
                torch.empty(H, D, device="cuda"))

    sets = [buffers() for _ in range(4)]
    torch.cuda.synchronize()
    for i in range(2):  # together
        run(i, *sets[i], streams[i])
    torch.cuda.synchronize()
    for i in range(2):  # one after the other
        run(i, *sets[2 + i], None)
        torch.cuda.synchronize()
        for a, b in ((0, 0), (4, 4), (5, 5)):
            assert torch.equal(sets[i][a], sets[2 + i][b])


def test_heads_and_rows_past_4_gib(attn):
    """A cache whose second KV head, and whose far rows, lie more than 4 GiB from its start."""
    ctx = 9_000_000
    g = gen(51)
    n = 100
    k, v = (torch.empty(KV, ctx, D, dtype=torch.float16, device="cuda") for _ in range(2))
    for t in (k, v):
        t[:, :n] = randn(g, KV, n, D, dtype=torch.float16)
    far = ctx - 200
    k[:, far:far + 8] = randn(g, KV, 8, D, dtype=torch.float16)
    v[:, far:far + 8] = randn(g, KV, 8, D, dtype=torch.float16)
    q, qg = 2.0 * randn(g, 5, H, D), randn(g, H, 2, D)
    w = torch.zeros(KV, ctx, device="cuda")
    added, rel = weights64(q, k[:, :n].double(), n - 5)
    attn.attn_prefill_weights(q, k, w, n - 5, 5, ctx, attn.PrefillWeightsScratch(5, n))
    zero = torch.zeros_like(w[:, :n])
    check(w[:, :n], zero, added, rel)
    w.zero_()
    attn.attn_decode_weights(q, qg, k, v, torch.empty(H, D, device="cuda"), w,
                             attn.DecodeWeightsScratch(128, n), n, ctx)
    added, rel = weights64(q[:1], k[:, :n].double(), n - 1)
    check(w[:, :n], zero, added, rel)
    assert (w[:, n:] == 0).all()
    w[:, far:far + 8] = torch.rand(KV, 8, generator=g, device="cuda") + 10
    index = torch.empty(KV, 12, dtype=torch.int32, device="cuda")
    attn.attn_evict_select(w, ctx, ctx, 12, 2, 2, index, attn.EvictScratch(ctx))
    want = [0, 1, *range(far, far + 8), ctx - 2, ctx - 1]
    assert index.tolist() == [want, want]
    v[:, ctx - 2:] = 1.0
    k[:, ctx - 2:] = 2.0
    ko, vo = (torch.zeros(KV, 12, D, dtype=torch.float16, device="cuda") for _ in range(2))
    wo = torch.zeros(KV, 12, device="cuda")
    attn.attn_evict_gather(k, v, w, ctx, index, 12, ko, vo, wo, 12)
    at = torch.tensor(want, device="cuda")
    assert torch.equal(ko, k[:, at]) and torch.equal(vo, v[:, at]) and torch.equal(wo, w[:, at])


def test_python_refusals(attn):
    f32 = dict(dtype=torch.float32, device="cuda")
    w, idx = torch.zeros(KV, 64, **f32), torch.zeros(KV, 8, dtype=torch.int32, device="cuda")
    q, qg, core = torch.zeros(H, D, **f32), torch.zeros(H, 2, D, **f32), torch.zeros(H, D, **f32)
    k = torch.zeros(KV, 64, D, dtype=torch.float16, device="cuda")
    sc, esc = attn.DecodeWeightsScratch(4, 32), attn.EvictScratch(32)
    psc = attn.PrefillWeightsScratch(4, 32)
    with pytest.raises(ValueError):  # beyond the scratch
        attn.attn_decode_weights(q, qg, k, k, core, w, sc, 33, 64)
    with pytest.raises(ValueError):
        attn.attn_decode_weights(q, qg, k, k, core, w, sc, 16, 64, n_splits=5)
    with pytest.raises(ValueError):
        attn.attn_decode_weights(q, qg, k, k, core, w[:, :32].contiguous(), sc, 16, 64)
    with pytest.raises(ValueError):
        attn.attn_decode_weights(q, qg, k, k, core, w.double(), sc, 16, 64)
    with pytest.raises(RuntimeError):
        attn.attn_decode_weights(q, qg, k, k, core, w, sc, 0, 64)
    with pytest.raises(ValueError):
        attn.attn_decode_weights(q, qg, k, k, core, w, sc, -1, 64)
    with pytest.raises(ValueError):
        attn.attn_prefill_weights(q, k, w, 0, 5, 64, psc)
    with pytest.raises(ValueError):
        attn.attn_prefill_weights(q, k, w, 31, 2, 64, psc)
    with pytest.raises(ValueError):
        attn.attn_prefill_weights(q, k, w, 0, 2, 64, psc)  # q holds one token
    with pytest.raises(ValueError):
        attn.attn_prefill_weights_fp8(q, attn.Fp8Cache(64), w, 0, 1, psc)
    with pytest.raises(ValueError):
        attn.attn_evict_select(w, 33, 64, 8, 0, 0, idx, esc)
    with pytest.raises(ValueError):
        attn.attn_evict_select(w, 32, 64, 9, 0, 0, idx, esc)
    with pytest.raises(ValueError):
        attn.attn_evict_select(w, 32, 64, 8, 0, 0, idx.long(), esc)
    with pytest.raises(RuntimeError):
        attn.attn_evict_select(w, 32, 64, 8, 5, 5, idx, esc)
    with pytest.raises(RuntimeError):  # in place
        attn.attn_evict_gather(k, k, w, 64, idx, 8, k, torch.empty_like(k), torch.empty_like(w), 64)
    with pytest.raises(ValueError):
        attn.attn_evict_gather(k, k, w, 64, idx, 8, k.int(), k.clone(), w.clone(), 64)
    with pytest.raises(ValueError):  # a host tensor
        attn.attn_evict_select(w.cpu(), 32, 64, 8, 0, 0, idx, esc)
