"""Decode behind a shared prefix on the GPU (no reference counterpart): paged and ragged against float64
over the same keys, at the decodes' precision, and a batch served from page plan to attention."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import REF_REL_L2
from test_shared_rule import rule

pytestmark = pytest.mark.gpu

H, KV, D, GROUP = 16, 2, 256, 8


def dev(torch, a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype or torch.int32).cuda()


def attention(torch, q, gate, k, v):
    """[16][256] in float64: one entry's gated attention over k, v [2][n][256]."""
    if k.shape[1] == 0:
        return torch.zeros(H, D, dtype=torch.float64, device="cuda")
    x = q.double().view(KV, GROUP, D)
    s = torch.matmul(x, k.double().transpose(1, 2).contiguous()) / 16
    return (torch.matmul(torch.softmax(s, -1), v.double()).view(H, D) *
            torch.sigmoid(gate.double()))


def check(torch, core, ref, what=""):
    err = (core.double() - ref).norm(dim=-1) / ref.norm(dim=-1).clamp(min=1e-300)
    err = torch.where(ref.abs().amax(-1) == 0, core.double().abs().amax(-1), err)
    assert torch.isfinite(core).all(), what
    assert err.max() <= REF_REL_L2, (what, float(err.max()))


class Paged:
    """Entries over a pool whose pages lie in random order; unused table entries and pages are bad."""

    def __init__(self, torch, page, prefix_pages, lens, seed, rows=None, q_scale=2.0, room=None):
        self.torch, self.page, self.pp = torch, page, prefix_pages
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.lens = np.asarray(lens)
        b = len(self.lens)
        self.rows = np.arange(b) if rows is None else np.asarray(rows)
        n_rows = int(self.rows.max()) + 1
        most = np.zeros(n_rows, np.int64)
        np.maximum.at(most, self.rows, np.maximum(self.lens - prefix_pages * page, 0))
        own = -(-most // page)
        self.room = room or prefix_pages + max(1, int(own.max()))
        total = prefix_pages + int(own.sum())
        ids = rng.permutation(total + 4)
        self.table = np.full((n_rows, self.room), -(2 ** 31) + 5, np.int64)
        at = prefix_pages
        for r in range(n_rows):
            self.table[r, :prefix_pages] = ids[:prefix_pages]
            self.table[r, prefix_pages:prefix_pages + own[r]] = ids[at:at + own[r]]
            at += own[r]
        self.prefix = ids[:prefix_pages]
        shape = (total + 4, KV, page, D)
        self.k = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)
        self.v = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)
        # Rows that nobody sees: the spare pages, and what lies behind a row's last key.
        for x in (self.k, self.v):
            x[torch.from_numpy(ids[total:]).cuda()] = float("nan")
            for r in range(n_rows):
                if own[r] and most[r] % page:
                    x[int(self.table[r, prefix_pages + own[r] - 1]), :, most[r] % page:] = (
                        float("inf"))
        self.q = q_scale * torch.randn(b, H, D, generator=g, device="cuda")
        self.gate = torch.randn(b, H, D, generator=g, device="cuda")
        self.core = torch.full((b, H, D), 777.25, device="cuda")
        self.max_own = int(most.max())
        self.d = dict(lens=dev(torch, self.lens), table=dev(torch, self.table),
                      prefix=dev(torch, self.prefix),
                      rows=None if rows is None else dev(torch, self.rows))

    def scratch(self, attn, **kw):
        sc = attn.SharedScratch(**{**dict(batch=len(self.lens), max_own=self.max_own,
                                          max_prefix=self.pp * self.page), **kw})
        sc.ws.fill_(255)  # NaN everywhere
        return sc

    def run(self, attn, sc=None, **kw):
        attn.attn_decode_paged_shared(self.q, self.gate, self.k, self.v, self.d["table"], self.page,
                                      self.d["lens"], self.d["prefix"], self.pp, self.core,
                                      sc or self.scratch(attn), rows=self.d["rows"], **kw)
        self.torch.cuda.synchronize()
        return self.core

    def keys(self, x, e):
        n, page = int(self.lens[e]), self.page
        table = self.table[self.rows[e]].copy()
        table[:self.pp] = self.prefix
        pages = self.torch.from_numpy(table[:-(-n // page)]).cuda()
        return x[pages].transpose(0, 1).reshape(KV, -1, D)[:, :n]

    def ref(self):
        return self.torch.stack([attention(self.torch, self.q[e], self.gate[e],
                                           self.keys(self.k, e), self.keys(self.v, e))
                                 for e in range(len(self.lens))])


def lengths(rng, batch, prefix, own, zeros=True):
    lens = prefix + rng.integers(0, own + 1, batch)
    if zeros and batch > 3:
        lens[rng.integers(0, batch)] = 0
        lens[rng.integers(0, batch)] = max(prefix // 2, 1)
        lens[rng.integers(0, batch)] = prefix
    lens[0] = prefix + own
    return lens


@pytest.mark.parametrize("batch,page,prefix_pages,own", [
    (1, 8, 1, 1), (1, 16, 40, 5), (2, 16, 0, 70), (3, 8, 3, 33), (4, 16, 130, 513), (5, 32, 1, 100),
    (7, 64, 9, 31), (8, 16, 17, 1030), (9, 8, 5, 8), (16, 128, 3, 300), (17, 16, 70, 64),
    (33, 16, 21, 700), (64, 8, 300, 129), (100, 256, 2, 40), (3, 4096, 1, 100), (20, 65536, 1, 9)])
def test_paged(torch_mod, attn, batch, page, prefix_pages, own):
    rng = np.random.default_rng(batch * 1000 + page)
    c = Paged(torch_mod, page, prefix_pages, lengths(rng, batch, prefix_pages * page, own), batch)
    first = c.run(attn).clone()
    check(torch_mod, first, c.ref())
    c.core.fill_(-5.0)
    assert torch_mod.equal(c.run(attn), first)  # the same bits over another dirty workspace


def test_paged_equals_the_paged_decode(torch_mod, attn):
    """The keys of attn_decode_paged on the same tables; entries without keys give zeros in both."""
    rng = np.random.default_rng(2)
    lens = lengths(rng, 21, 320, 300)
    c = Paged(torch_mod, 16, 20, lens, 21)
    c.d["table"].clamp_(min=0)  # (that call reads no bad entry either, but says so of fewer)
    got = c.run(attn).clone()
    other = torch_mod.empty_like(got)
    attn.attn_decode_paged(c.q, c.gate, c.k, c.v, c.d["table"], 16, c.d["lens"], other,
                           attn.RaggedScratch(21, int(lens.max())))
    check(torch_mod, got, other.double())
    empty = torch_mod.from_numpy(lens == 0).cuda()
    assert (got[empty] == 0).all() and empty.any()


@pytest.mark.parametrize("batch,seqs,prefix_pages", [(6, 1, 2), (40, 1, 30), (203, 1, 12),
                                                     (24, 3, 5), (9, 2, 0)])
def test_chunks_share_a_table_row(torch_mod, attn, batch, seqs, prefix_pages):
    """Entries of one row with rising lengths: the causal attention of a chunk of each request."""
    page = 16
    rows = np.arange(batch) * seqs // batch
    count = np.bincount(rows)
    index = np.arange(batch) - np.concatenate([[0], np.cumsum(count)])[rows]
    lens = prefix_pages * page + 11 * rows + index + 1
    c = Paged(torch_mod, page, prefix_pages, lens, batch, rows=rows)
    check(torch_mod, c.run(attn), c.ref())


@pytest.mark.parametrize("batch,own", [(513, 40), (1100, 5), (600, 700)])
def test_many_entries(torch_mod, attn, batch, own):
    """Above the entries of one streaming launch."""
    rng = np.random.default_rng(batch)
    c = Paged(torch_mod, 16, 3, lengths(rng, batch, 48, own), batch)
    check(torch_mod, c.run(attn), c.ref())


def test_many_entries_of_few_rows(torch_mod, attn):
    """Chunks of two requests, more entries than one streaming launch takes."""
    rows = np.arange(700) // 400
    lens = 64 + 1 + np.arange(700) % 400
    c = Paged(torch_mod, 16, 4, lens, 700, rows=rows)
    check(torch_mod, c.run(attn), c.ref())


def test_thousands_of_entries(torch_mod, attn):
    """More row groups than CUs; some entries against float64, those of equal queries against each other."""
    torch = torch_mod
    rng = np.random.default_rng(3)
    lens = lengths(rng, 9000, 64, 3)
    c = Paged(torch, 16, 4, lens, 9000)
    c.core = torch.full((9002, H, D), 777.25, device="cuda")
    got = c.run(attn)
    assert (got[9000:] == 777.25).all()  # behind the last entry
    for e in [0, 1, 2047, 2048, 4095, 4096, 8191, 8192, 8999, *rng.integers(0, 9000, 40)]:
        ref = attention(torch, c.q[e], c.gate[e], c.keys(c.k, e), c.keys(c.v, e))
        check(torch, got[e][None], ref[None], e)
    assert (got[:9000][torch.from_numpy(lens == 0).cuda()] == 0).all()


def test_own_keys_beyond_max_own(torch_mod, attn):
    """lens above the capacity the scratch was made for: still all keys, in longer spans."""
    c = Paged(torch_mod, 8, 4, [32 + 2049, 32 + 5, 32], 3)
    sc = c.scratch(attn, max_own=600)
    check(torch_mod, c.run(attn, sc), c.ref())


def test_max_own_of_zero_looks_at_the_prefix_alone(torch_mod, attn):
    c = Paged(torch_mod, 8, 6, [48, 48, 20, 0, 48], 4, room=6)
    c.table[:] = -1
    check(torch_mod, c.run(attn, c.scratch(attn, max_own=0)), c.ref())


def test_scratch_serves_smaller_calls(torch_mod, attn):
    rng = np.random.default_rng(8)
    sc = attn.SharedScratch(64, 900, 4096)
    for batch, pp, own in ((64, 256, 900), (1, 256, 900), (13, 3, 40), (64, 1, 1), (9, 255, 700)):
        c = Paged(torch_mod, 16, pp, lengths(rng, batch, 16 * pp, own), batch)
        check(torch_mod, c.run(attn, sc), c.ref(), (batch, pp, own))


@pytest.mark.parametrize("batch", [2, 7, 16, 17])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 6, 7, 12])
def test_every_count_of_tiles_in_a_span(torch_mod, attn, batch, tiles):
    """The streaming loop's start, ring and end, by one, two and four row blocks a workgroup (128 spans,
    64 for 17 entries), the last span shorter."""
    keys = tiles * 32 * (128 if batch <= 16 else 64) - 24
    c = Paged(torch_mod, 8, keys // 8, [keys + 1 if e % 3 else keys - 5 * e for e in range(batch)],
              tiles)
    check(torch_mod, c.run(attn), c.ref())


@pytest.mark.parametrize("batch,prefix_pages", [(3, 300), (7, 300), (24, 128), (150, 600), (490, 160)])
def test_cut_by_the_lengths(torch_mod, attn, batch, prefix_pages):
    """A scratch for 4000 own keys and batches that have far fewer, or nearly those: the CUs of the prefix
    and of the own keys, and the spans with them, follow the lengths; one scratch serves all."""
    rng = np.random.default_rng(batch)
    sc = None
    for own in (0, 1, 40, 300, 3990 if batch < 100 else 900):
        c = Paged(torch_mod, 16, prefix_pages, lengths(rng, batch, 16 * prefix_pages, own), batch,
                  room=prefix_pages + 250)
        sc = sc or c.scratch(attn, max_own=4000)
        first = c.run(attn, sc).clone()
        check(torch_mod, first, c.ref(), own)
        sc.ws.fill_(255)
        assert torch_mod.equal(c.run(attn, sc), first), own


@pytest.mark.parametrize("batch", [63, 64, 130, 512])
@pytest.mark.parametrize("own", [1, 33, 256, 257])
def test_few_own_keys(torch_mod, attn, batch, own):
    """Around the lengths and batches whose own keys are a wave's each, paged and ragged; one workspace for
    rising and falling lengths."""
    torch = torch_mod
    rng = np.random.default_rng(batch + own)
    for pp in (4, 90):
        lens = 16 * pp + rng.choice([0, 1, 31, 32, 33, own, rng.integers(0, own + 1)], batch)
        lens = np.minimum(lens, 16 * pp + own)
        lens[5], lens[6] = 0, 16 * pp + own
        c = Paged(torch, 16, pp, lens, batch)
        sc = c.scratch(attn, max_own=2000 if own == 33 else own)
        check(torch, c.run(attn, sc), c.ref(), pp)
    r = ragged(torch, batch, 300, own, own)
    core, ref = run_ragged(torch, attn, r)
    check(torch, core, ref)


@pytest.mark.parametrize("batch,prefix,max_own", [(8, 32768, 7988), (8, 16384, 4096),
                                                  (16, 32768, 1024), (24, 8192, 1024)])
def test_no_own_keys_leave_no_workgroup_for_them(torch_mod, attn, batch, prefix, max_own):
    """The kernel gives the whole launch to the prefix, so that nobody chooses the own keys' span: over a
    workspace of zeros, of ones and of an earlier call's words, and with own keys again after it."""
    c = Paged(torch_mod, 16, prefix // 16, [prefix] * (batch - 2) + [0, prefix - 100], batch,
              room=prefix // 16 + -(-max_own // 16))
    sc = c.scratch(attn, max_own=max_own)
    ref = c.ref()
    for fill in (0, 255, 1):
        sc.ws.fill_(fill)
        c.core.fill_(777.25)
        check(torch_mod, c.run(attn, sc), ref, fill)
    other = Paged(torch_mod, 16, prefix // 16, [prefix + 90 + 31 * e for e in range(batch)], batch)
    check(torch_mod, other.run(attn, sc), other.ref())
    c.core.fill_(777.25)
    check(torch_mod, c.run(attn, sc), ref)


def test_spans_longer_than_the_page_ids_a_wave_holds(torch_mod, attn):
    """More than 64 tiles a span: its pages are read again, and tiles wrap the ring many times."""
    lens = 90112 + np.arange(30) % 7
    lens[3] = 50001  # ends inside a span
    c = Paged(torch_mod, 16, 5632, lens, 30)
    check(torch_mod, c.run(attn), c.ref())


def test_extreme_scores(torch_mod, attn):
    """Queries of 2^-20 .. 2^16 (2^20 over the prefix alone: the split over own keys takes those below
    2^19) and rising keys: references move late in a span, weights of 0 and 1."""
    torch = torch_mod
    for scale, own in ((2.0 ** -20, 90), (30.0, 90), (2.0 ** 16, 90), (2.0 ** 20, 0)):
        c = Paged(torch, 16, 16, lengths(np.random.default_rng(1), 19, 256, own, zeros=False), 6,
                  q_scale=scale)
        if scale == 30.0:
            ramp = torch.linspace(0.01, 1.5, 256, device="cuda", dtype=torch.float16)
            pages = torch.from_numpy(c.prefix).cuda()
            c.k[pages] = (c.k[pages].transpose(1, 2) * ramp.view(16, 16, 1, 1)).transpose(1, 2)
        got, ref = c.run(attn), c.ref()
        # A score s is off by 2^-22 of |q| |k| / 16 (pairs) and 2^-23 (sums), its weight by that factor.
        if scale <= 30.0:
            size = float(c.q.norm(dim=-1).max()) * float(c.k[~c.k.isnan() & ~c.k.isinf()].abs().max())
            err = ((got.double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
            assert err <= REF_REL_L2 + 2.0 ** -21 * size, float(err)
        else:  # one key has all the weight, unless two scores lie within rounding
            assert torch.isfinite(got).all()
            assert ((got.double() - ref).norm(dim=-1) <= 1e-4 * ref.norm(dim=-1)).float().mean() > 0.98


@pytest.mark.parametrize("b", [70, 12])  # own keys a wave's each, or by four waves
@pytest.mark.parametrize("top", [500, 2000, 16000])
def test_equal_scores_of_a_prefix_key_and_an_own_key_weigh_evenly(torch_mod, attn, top, b):
    """One key of the prefix and one of the entry's own with the same large score, the others at 0: half the
    weight each. Queries have one element, and that times log2(e) has 21 significant bits, so that both sides
    hold the score exactly; what is left are the sums' and the gate's roundings, far below the 1e-5. (To natural
    units and back a reference in [2^k, 2^(k+1)) moves by up to 2^(k-24).)"""
    torch = torch_mod
    rng = np.random.default_rng(top)
    log2e = np.float32(1.4426950408889634)

    def query():
        while True:
            t = top / 2 * (1 + rng.random())  # score 2 t in log2 units
            t = np.round(t * 2.0 ** (20 - int(np.floor(np.log2(t))))) * 2.0 ** -(
                20 - int(np.floor(np.log2(t))))
            q = np.float32(t / np.float64(log2e))
            if np.float32(q * log2e) == t:
                return q

    own = 40
    c = Paged(torch, 16, 4, [64 + own - e % 5 for e in range(b)], 3)
    finite = torch.isfinite(c.k)
    c.k.mul_(torch.where(finite, 0, 1).half())  # 0, and NaN and infinity where nobody sees
    c.q.zero_()
    c.q[:, :, 0] = torch.from_numpy(np.array([[query() for _ in range(H)] for _ in range(b)])).cuda()
    for e in range(b):
        for key in (rng.integers(0, 64), rng.integers(64, c.lens[e])):
            page = c.prefix[key // 16] if key < 64 else c.table[e, key // 16]
            if key >= 64 or e == 0:  # one key of the prefix
                c.k[int(page), :, int(key) % 16, 0] = 32
    check(torch, c.run(attn), c.ref())
    # The same behind a contiguous prefix.
    r = ragged(torch, b, 64, own, top)
    r["held"][:] = own
    r["first"] = np.arange(b) * KV * own * D
    rand = lambda *n: torch.randn(*n, device="cuda", dtype=torch.float16)  # noqa: E731
    r["k"], r["v"] = torch.zeros(b * KV * own * D, device="cuda").half(), rand(b * KV * own * D)
    r["k"].view(b, KV, own, D)[:, :, 17, 0] = 32
    r["kp"][:, :64] = 0
    r["kp"][:, 29, 0] = 32
    r["q"] = c.q
    core, ref = run_ragged(torch, attn, r)
    check(torch, core, ref)


@pytest.mark.parametrize("q_scale", [0.01, 1.0, 4.0])
@pytest.mark.parametrize("batch", [3, 7, 19, 70])
def test_precision_of_ordinary_scores(torch_mod, attn, batch, q_scale):
    """1e-5 while no key's sum of |q_i k_i| / 16 exceeds 64 (about 54 here at most)."""
    c = Paged(torch_mod, 16, 130, lengths(np.random.default_rng(batch), batch, 2080, 400), batch,
              q_scale=q_scale)
    for e in range(min(batch, 8)):
        size = torch_mod.matmul(c.q[e].abs().view(KV, GROUP, D),
                                c.keys(c.k, e).float().abs().transpose(1, 2).contiguous()) / 16
        assert size.numel() == 0 or size.max() <= 64
    check(torch_mod, c.run(attn), c.ref())


def test_rows_are_independent(torch_mod, attn):
    """NaN and infinities in the queries of an entry stay in its rows; queries of zero weigh evenly."""
    torch = torch_mod
    c = Paged(torch, 16, 10, lengths(np.random.default_rng(4), 18, 160, 60, zeros=False), 18)
    c.q[5] = 0
    good = c.run(attn).clone()
    check(torch, good, c.ref())
    c.q[3] = float("nan")
    c.q[7, 2] = float("inf")
    c.q[12] = 3e38
    got = c.run(attn)
    keep = torch.ones(18, H, dtype=torch.bool, device="cuda")
    keep[3] = keep[12] = keep[7, 2] = False
    assert torch.equal(got[keep], good[keep])


@pytest.mark.parametrize("batch,prefix_pages,most", [
    (1, 4, 1), (1, 40, 613), (3, 300, 4799), (4, 64, 31), (7, 300, 4000), (8, 20, 0), (16, 40, 300),
    (20, 300, 1025), (40, 300, 4769), (70, 9, 143), (520, 5, 33), (520, 5, 79)])
def test_rows_of_the_prefix_that_nobody_sees_may_hold_anything(torch_mod, attn, batch, prefix_pages, most):
    """Entries that all end inside the prefix, as the paged decode serves them: behind the longest's keys lie NaN
    and infinities, in K and in V; an entry of length 0 sees none."""
    torch, page = torch_mod, 16
    rng = np.random.default_rng(batch + most)
    lens = rng.integers(0, most + 1, batch)
    lens[rng.integers(0, batch)] = most
    c = Paged(torch, page, prefix_pages, lens, batch + most)
    clean = c.run(attn).clone()
    check(torch, clean, c.ref())
    ids = torch.from_numpy(c.prefix).cuda()
    for x, bad in ((c.k, float("nan")), (c.v, float("inf")), (c.v, float("nan")), (c.k, float("-inf"))):
        rows = x[ids].transpose(0, 1).reshape(KV, -1, D)
        rows[:, most:] = bad
        x[ids] = rows.view(KV, prefix_pages, page, D).transpose(0, 1).contiguous()
        c.core.fill_(777.25)
        assert torch.equal(c.run(attn), clean)
    assert torch.isfinite(clean).all()


def test_unseen_rows_beside_entries_behind_the_prefix(torch_mod, attn):
    """Row groups of their own: entries 0 .. 31 end inside the prefix at 700 or before, the last one sees up to
    1100 of 1600 rows; the rows behind hold NaN."""
    torch = torch_mod
    rng = np.random.default_rng(5)
    lens = np.concatenate([rng.integers(0, 701, 32), [1100]])
    c = Paged(torch, 16, 100, lens, 9)
    clean = c.run(attn).clone()
    check(torch, clean, c.ref())
    for x in (c.k, c.v):
        x[torch.from_numpy(c.prefix[70:]).cuda()] = float("nan")
        x[int(c.prefix[68]), :, 12:] = float("nan")
        x[int(c.prefix[69])] = float("inf")
    assert torch.equal(c.run(attn), clean)


def test_padding_entries_read_nothing(torch_mod, attn):
    """Entries of length 0 with NaN queries, rows outside the table's use: zeros, the others whole."""
    torch = torch_mod
    lens = np.array([200, 0, 0, 161, 0, 160, 190, 0, 0, 0])
    c = Paged(torch, 16, 10, lens, 5, rows=np.array([0, 0, 0, 1, 0, 2, 3, 0, 0, 0]))
    ref = c.ref()
    for e in np.flatnonzero(lens == 0):
        c.q[e] = float("nan")
        c.d["rows"][int(e)] = 2 ** 30
    got = c.run(attn)
    check(torch, got, ref)
    assert (got[torch.from_numpy(lens == 0).cuda()] == 0).all()


def test_pool_beyond_4_gib(torch_mod, attn):
    torch, page, pp = torch_mod, 64, 20
    c = Paged(torch, page, pp, [pp * page + 100, pp * page + 7, pp * page], 31)
    pages = 80000  # 5.2 GB each
    far = np.random.default_rng(1).permutation(4000)[:len(c.k)] + pages - 4000
    k, v = (torch.empty(pages, KV, page, D, device="cuda", dtype=torch.float16) for _ in range(2))
    at = torch.from_numpy(far).cuda()
    k[at], v[at] = c.k, c.v
    ref = c.ref()
    table = np.where(c.table >= 0, far[np.clip(c.table, 0, len(far) - 1)], -1)
    c.k, c.v = k, v
    c.d["table"], c.d["prefix"] = dev(torch, table), dev(torch, far[c.prefix])
    check(torch, c.run(attn), ref)


def ragged(torch, batch, prefix, own, seed, ctx_spare=13):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    held = rng.integers(0, own + 1, batch)
    held[0] = own
    first = np.concatenate([[0], np.cumsum(held)[:-1]]) * KV * D
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    total, ctx = max(int(held.sum()), 1), prefix + ctx_spare
    c = dict(held=held, q=2 * torch.randn(batch, H, D, generator=g, device="cuda"),
             gate=torch.randn(batch, H, D, generator=g, device="cuda"), k=rand(total * KV * D),
             v=rand(total * KV * D), kp=rand(KV, ctx, D), vp=rand(KV, ctx, D), first=first,
             prefix=prefix, ctx=ctx, core=torch.full((batch, H, D), -3.5, device="cuda"))
    c["kp"][:, prefix:], c["vp"][:, prefix:] = float("nan"), float("inf")
    return c


def run_ragged(torch, attn, c, sc=None):
    sc = sc or attn.SharedScratch(len(c["held"]), int(c["held"].max()), c["prefix"])
    attn.attn_decode_ragged_shared(c["q"], c["gate"], c["k"], c["v"],
                                   dev(torch, c["first"], torch.int64), dev(torch, c["held"]),
                                   c["kp"], c["vp"], c["prefix"], c["ctx"], c["core"], sc)
    ref = []
    for e, n in enumerate(c["held"]):
        n, at = int(n), int(c["first"][e])
        kv = [torch.cat([p[:, :c["prefix"]], x[at:at + KV * n * D].view(KV, n, D)], dim=1)
              for p, x in ((c["kp"], c["k"]), (c["vp"], c["v"]))]
        ref.append(attention(torch, c["q"][e], c["gate"][e], *kv))
    return c["core"], torch.stack(ref)


@pytest.mark.parametrize("batch,prefix,own", [
    (1, 1, 0), (1, 31, 3), (2, 32, 40), (3, 33, 1), (4, 1000, 600), (6, 257, 10), (8, 4097, 64),
    (13, 65, 900), (16, 0, 50), (33, 5003, 100), (70, 511, 17), (530, 63, 9)])
def test_ragged(torch_mod, attn, batch, prefix, own):
    c = ragged(torch_mod, batch, prefix, own, batch + prefix)
    core, ref = run_ragged(torch_mod, attn, c)
    check(torch_mod, core, ref)


def test_ragged_without_a_prefix_takes_none(torch_mod, attn):
    """prefix_len 0: the prefix's caches are not looked at, whether None or anything else."""
    c = ragged(torch_mod, 5, 0, 70, 2)
    core, ref = run_ragged(torch_mod, attn, c)
    check(torch_mod, core, ref)
    first = core.clone()
    sc = attn.SharedScratch(5, 70, 0)
    args = (c["q"], c["gate"], c["k"], c["v"], dev(torch_mod, c["first"], torch_mod.int64),
            dev(torch_mod, c["held"]))
    for none in (None, torch_mod.zeros(3)):
        core.fill_(777.25)
        attn.attn_decode_ragged_shared(*args, none, none, 0, 0, core, sc)
        assert torch_mod.equal(core, first)
    with pytest.raises(ValueError, match="k_prefix"):
        attn.attn_decode_ragged_shared(*args, torch_mod.zeros(3), torch_mod.zeros(3), 1, 1, core,
                                       attn.SharedScratch(5, 70, 1))


@pytest.mark.parametrize("prefix", [0, 100])
def test_ragged_of_empty_caches(torch_mod, attn, prefix):
    """No sequence has own keys, the caches are empty, the scratch is made for more: the prefix alone."""
    c = ragged(torch_mod, 5, prefix, 0, 2)
    c["k"], c["v"] = c["k"][:0], c["v"][:0]
    core, ref = run_ragged(torch_mod, attn, c, attn.SharedScratch(6, 300, 128))
    check(torch_mod, core, ref)


def test_ragged_prefix_beyond_4_gib(torch_mod, attn):
    """A cache of 4.3 million rows a head: the second head's rows lie past 32-bit byte and half offsets."""
    torch = torch_mod
    c = ragged(torch, 5, 700, 20, 3)
    ctx = 9_000_000  # 4.6 GB a head
    for x in ("kp", "vp"):
        far = torch.empty(KV, ctx, D, device="cuda", dtype=torch.float16)
        far[:, :700] = c[x][:, :700]
        c[x] = far
    c["ctx"] = ctx
    core, ref = run_ragged(torch, attn, c)
    check(torch, core, ref)


def test_two_streams_and_graphs(torch_mod, attn):
    """Two calls at once over scratches of their own, and a captured call replayed over new lengths."""
    torch = torch_mod
    a = Paged(torch, 16, 40, lengths(np.random.default_rng(1), 12, 640, 200), 1)
    b = Paged(torch, 8, 9, lengths(np.random.default_rng(2), 40, 72, 90), 2)
    sa, sb = a.scratch(attn), b.scratch(attn)
    ra, rb = a.run(attn, sa).clone(), b.run(attn, sb).clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        a.core.zero_()
        b.core.zero_()
        torch.cuda.synchronize()
        for c, sc, s in ((a, sa, streams[0]), (b, sb, streams[1])):
            attn.attn_decode_paged_shared(c.q, c.gate, c.k, c.v, c.d["table"], c.page, c.d["lens"],
                                          c.d["prefix"], c.pp, c.core, sc, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(a.core, ra) and torch.equal(b.core, rb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.attn_decode_paged_shared(a.q, a.gate, a.k, a.v, a.d["table"], a.page, a.d["lens"],
                                      a.d["prefix"], a.pp, a.core, sa)
    for step in range(4):
        a.lens = np.minimum(lengths(np.random.default_rng(step), 12, 640, 200), a.lens)
        a.d["lens"].copy_(dev(torch, a.lens))
        a.q.normal_()
        sa.ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        check(torch, a.core, a.ref(), step)


def test_two_graphs_share_a_workspace(torch_mod, attn):
    """Calls of different batches, prefixes and lengths captured over one scratch, replayed in turn with eager
    work between."""
    torch = torch_mod
    cases = [Paged(torch, 16, 200, lengths(np.random.default_rng(1), 9, 3200, 700), 1),
             Paged(torch, 8, 5, lengths(np.random.default_rng(2), 90, 40, 30), 2),
             Paged(torch, 32, 40, lengths(np.random.default_rng(3), 30, 1280, 500), 3)]
    sc = attn.SharedScratch(90, 1000, 3200)
    graphs, refs = [], []
    for c in cases:
        c.run(attn, sc)
        refs.append(c.core.clone())
        check(torch, c.core, c.ref())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attn.attn_decode_paged_shared(c.q, c.gate, c.k, c.v, c.d["table"], c.page, c.d["lens"],
                                          c.d["prefix"], c.pp, c.core, sc)
        graphs.append(graph)
    for i in (0, 1, 2, 1, 0, 2, 2, 0, 1):
        cases[i].core.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(cases[i].core, refs[i]), i
        sc.ws[::7].add_(1)


def test_a_batch_served(torch_mod, attn):
    """Steps of a server: plan, prep and attention over one pool, requests behind a shared prefix that
    start with prompts, go on by one token and end; every step's outputs against float64 over the keys
    that the prep wrote, and the keys against a record of what each request was given."""
    torch = torch_mod
    rng = np.random.default_rng(21)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    b, page, pp, room, pool, most = 12, 8, 6, 20, 170, 96
    stride = 9216
    k_pages, v_pages = (torch.zeros(pool, KV, page, D, device="cuda", dtype=torch.float16)
                        for _ in range(2))
    ids = rng.permutation(pool)
    prefix = dev(torch, ids[:pp])
    k_pages[prefix.long()] = torch.randn(pp, KV, page, D, generator=g, device="cuda").half()
    v_pages[prefix.long()] = torch.randn(pp, KV, page, D, generator=g, device="cuda").half()
    lens, table = dev(torch, np.zeros(b)), dev(torch, np.full((b, room), -1))
    stack, n_free = dev(torch, np.concatenate([ids[pp:], np.full(pp, -1)])), dev(torch, [pool - pp])
    q_norm, k_norm = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    freq, scale = attn.rope_frequencies(64, 1e7, factor=4, scaling="yarn", original_ctx=32768)
    plan = attn.PagePlan(b, most)
    q, gate, core = (torch.full((most, H, D), 5.0, device="cuda") for _ in range(3))
    sc = attn.SharedScratch(most, (room - pp) * page, pp * page)
    given = [[] for _ in range(b)]  # per request: (step, token) of its keys behind the prefix
    projs = []
    held = np.zeros(b, np.int64)
    for step in range(9):
        ended = (rng.random(b) < 0.15) & (held > 0)
        new = np.where(held == 0, rng.integers(0, 15, b), 1)
        new[ended] = rng.integers(0, 2, b)[ended] * 9
        proj = torch.randn(most, stride, generator=g, device="cuda")
        projs.append(proj)
        attn.attn_page_plan(lens, dev(torch, new), table, page, stack, n_free, plan,
                            ended=dev(torch, ended), prefix_table=prefix, prefix_pages=pp)
        flat = proj.view(-1)
        attn.attn_prep_paged(flat, flat[8192:], flat[8704:], q_norm, k_norm, freq, k_pages, v_pages,
                             page, plan.slots, plan.positions, q, most, stride, 1e-6, gate=gate,
                             rot_scale=scale)
        attn.attn_decode_paged_shared(q, gate, k_pages, v_pages, table, page, plan.visible, prefix,
                                      pp, core, sc, rows=plan.rows)
        torch.cuda.synchronize()
        status, starts = plan.status.cpu().numpy(), plan.starts.cpu().numpy()
        for r in range(b):
            if ended[r]:
                given[r], held[r] = [], 0
            if new[r] and status[r] == 0:
                given[r] += [(step, t) for t in range(starts[r], starts[r + 1])]
                held[r] = pp * page + len(given[r])
        assert np.array_equal(lens.cpu().numpy(), held)
        rows, sees = plan.rows.cpu().numpy(), plan.visible.cpu().numpy()
        t_of = table.cpu().numpy()
        for t in range(most):
            if sees[t] == 0:
                assert (core[t] == 0).all()
                continue
            pages = torch.from_numpy(np.concatenate([ids[:pp], t_of[rows[t]][pp:]])[
                :-(-sees[t] // page)]).cuda().long()
            k = k_pages[pages].transpose(0, 1).reshape(KV, -1, D)[:, :sees[t]]
            v = v_pages[pages].transpose(0, 1).reshape(KV, -1, D)[:, :sees[t]]
            check(torch, core[t][None], attention(torch, q[t], gate[t], k, v)[None], (step, t))
            if t == starts[rows[t] + 1] - 1:  # V rows are the given tokens', in order
                mine = torch.stack([projs[s][i, 8704:].view(KV, D) for s, i in given[rows[t]]], 1)
                assert torch.equal(v[:, pp * page:], mine.half())
    assert held.max() > 0


def last_span(r, tiles):
    """Tiles of the last span of a rule."""
    return tiles - (r["spans"] - 1) * r["span_tiles"]


@pytest.mark.parametrize("batch,row_blocks", [(3, 1), (7, 2), (12, 2), (515, 4)])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 6, 7])
def test_spans_of_every_few_tiles(torch_mod, attn, O, batch, row_blocks, tiles):
    """One span of 1 .. 7 tiles, whole and ending inside a tile, by one, two and four row blocks a workgroup:
    the ring's first copies, none and some left to issue in the loop. (Spans that the cut makes several of have
    4 tiles and more, but the last one; see below.)"""
    for page, cut in ((8, 0), (8, 24), (32, 0)):
        keys = 32 * tiles - cut
        r = rule(O, batch, keys, 0)
        assert (r["row_blocks"], r["spans"], r["span_tiles"]) == (row_blocks, 1, tiles)
        lens = np.array([max(keys - 5 * (e % 4), 0) for e in range(batch)])
        c = Paged(torch_mod, page, keys // page, lens, batch + tiles)
        check(torch_mod, c.run(attn, c.scratch(attn, max_own=0)), c.ref(), (page, cut))


@pytest.mark.parametrize("batch,row_blocks", [(4, 1), (8, 2), (300, 4)])
@pytest.mark.parametrize("last", [1, 2, 3, 4, 5])
def test_last_spans_of_every_few_tiles(torch_mod, attn, O, batch, row_blocks, last):
    """A last span of 1 .. 5 tiles behind longer ones, its last tile of one row, of 31 and whole."""
    def fits(tiles, off):
        r = rule(O, batch, 32 * tiles - off, 0)
        return r["row_blocks"] == row_blocks and r["spans"] > 1 and last_span(r, tiles) == last

    for off in (0, 1, 31):
        tiles = next(t for t in range(5, 4000) if fits(t, off))
        c = ragged(torch_mod, batch, 32 * tiles - off, 0, tiles)
        core, ref = run_ragged(torch_mod, attn, c, attn.SharedScratch(batch, 0, c["prefix"]))
        check(torch_mod, core, ref, (tiles, off))


@pytest.mark.parametrize("q_scale,own", [(30.0, 90), (300.0, 90), (2.0 ** 13, 90), (2.0 ** 16, 90),
                                         (2.0 ** 20, 0)])
@pytest.mark.parametrize("batch", [3, 19, 70])
def test_every_head_of_large_scores(torch_mod, attn, batch, q_scale, own):
    """A score is off by at most d = 2^-17.8 of the sum of its |q_i k_i| / 16: queries as pairs 2^-21, log2(e)
    and its product 2^-24 and 2^-25, 32 sums in f32 of 2^-23 at most (rounded or cut), 2^-18 of them. With the
    largest such d over a head's keys, D, a weight is off by a factor of up to e^(2 D): the output by
    (e^(2 D) - 1) sum w |v|. Where a key leads by more than 2 D + 20, the others weigh less than n e^-20, 2e-7
    here, and the output is that key's value to the decodes' 1e-5. What is left are heads between: those lie
    within the values."""
    torch = torch_mod
    c = Paged(torch, 16, 16, lengths(np.random.default_rng(batch), batch, 256, own), batch + 1,
              q_scale=q_scale)
    got = c.run(attn).double()
    assert torch.isfinite(got).all()
    held = heads = 0
    for e in np.flatnonzero(c.lens):
        k, v = c.keys(c.k, e).double(), c.keys(c.v, e).double()
        q = c.q[e].double().view(KV, GROUP, D)
        kt = k.transpose(1, 2).contiguous()
        d = 2.0 ** -17.8 * (torch.matmul(q.abs(), kt.abs()) / 16).amax(-1)
        s = torch.matmul(q, kt) / 16
        w = torch.softmax(s, -1)
        gate = torch.sigmoid(c.gate[e].double()).view(KV, GROUP, D)
        ref, out = torch.matmul(w, v) * gate, got[e].view(KV, GROUP, D)
        err, norm = (out - ref).norm(dim=-1), ref.norm(dim=-1)
        spread = torch.matmul(w, v.norm(dim=-1, keepdim=True))[..., 0]
        near = torch.expm1((2 * d).clamp(max=50.0)) * spread + REF_REL_L2 * norm
        if s.shape[-1] > 1:
            top = s.topk(2, dim=-1).values
            leads = top[..., 0] - top[..., 1] > 2 * d + 20
        else:
            leads = torch.ones_like(norm, dtype=torch.bool)
        bound = torch.where(leads, REF_REL_L2 * norm, near)
        assert (err <= bound).all(), (int(e), float((err / bound).max()))
        assert (out.abs() <= v.abs().amax(1)[:, None] * gate * (1 + 1e-5) + 1e-30).all()
        held += int((bound <= 0.2 * norm).sum())
        heads += norm.numel()
    assert held >= 0.98 * heads, (held, heads)  # the bound says something of nearly all


@pytest.mark.parametrize("capacity,live,prefix_pages,own", [(512, 64, 64, 300), (300, 1, 40, 30),
                                                            (2000, 33, 16, 50), (64, 5, 400, 1)])
def test_empty_entries_behind_the_live_ones(torch_mod, attn, capacity, live, prefix_pages, own):
    """A step's capacity of which most is empty at the end, NaN queries there: zeros, the live ones whole."""
    torch = torch_mod
    lens = np.zeros(capacity, np.int64)
    lens[:live] = lengths(np.random.default_rng(live), live, 16 * prefix_pages, own, zeros=False)
    c = Paged(torch, 16, prefix_pages, lens, capacity)
    ref = c.ref()
    c.q[live:] = float("nan")
    for _ in range(2):
        c.core.fill_(777.25)
        got = c.run(attn)
        check(torch, got, ref)
        assert (got[live:] == 0).all()


@pytest.mark.parametrize("prefix_pages", [0, 10])
def test_empty_entries_give_zeros_whatever_their_gates_hold(torch_mod, attn, prefix_pages):
    """attn_prep_paged leaves the gates of tokens without a slot as they are: NaN, where nobody wrote them."""
    torch = torch_mod
    lens = np.array([0, 16 * prefix_pages + 40, 0, 16 * prefix_pages + 1, 0, 0])
    c = Paged(torch, 16, prefix_pages, lens, 5)
    ref = c.ref()
    for bad in (float("nan"), float("inf"), -float("inf")):
        c.gate[torch.from_numpy(lens == 0).cuda()] = bad
        c.core.fill_(777.25)
        check(torch, c.run(attn), ref)
    r = ragged(torch, 4, 0, 30, 6)
    r["held"][1:3] = 0
    core, ref = run_ragged(torch, attn, r)
    check(torch, core, ref)
    r["gate"][1:3] = float("nan")
    run_ragged(torch, attn, r)
    check(torch, r["core"], ref)


def test_a_plan_of_large_capacity(torch_mod, attn):
    """attn_page_plan's rows and visible for 512 tokens of which 40 are given, as one call's entries."""
    torch = torch_mod
    rng = np.random.default_rng(1)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    b, page, pp, room, pool, most = 30, 16, 50, 60, 400, 512
    ids = rng.permutation(pool)
    rand = lambda *n, **kw: torch.randn(*n, generator=g, device="cuda", **kw)  # noqa: E731
    k, v = (rand(pool, KV, page, D, dtype=torch.float16) for _ in range(2))
    prefix, table = dev(torch, ids[:pp]), dev(torch, np.full((b, room), -1))
    lens, stack = dev(torch, np.zeros(b)), dev(torch, np.concatenate([ids[pp:], np.full(pp, -1)]))
    n_free, plan = dev(torch, [pool - pp]), attn.PagePlan(b, most)
    new = np.ones(b, np.int64)
    new[3] = 11  # a chunk among single tokens
    attn.attn_page_plan(lens, dev(torch, new), table, page, stack, n_free, plan,
                        prefix_table=prefix, prefix_pages=pp)
    q, gate = 2 * rand(most, H, D), rand(most, H, D)
    core = torch.full((most, H, D), 5.0, device="cuda")
    sc = attn.SharedScratch(most, (room - pp) * page, pp * page)
    sc.ws.fill_(255)
    attn.attn_decode_paged_shared(q, gate, k, v, table, page, plan.visible, prefix, pp, core, sc,
                                  rows=plan.rows)
    torch.cuda.synchronize()
    rows, sees, t_of = (x.cpu().numpy() for x in (plan.rows, plan.visible, table))
    assert (sees[:40] > pp * page).all() and (sees[40:] == 0).all() and new.sum() == 40
    assert (core[40:] == 0).all()
    for t in range(40):
        pages = torch.from_numpy(t_of[rows[t]][:-(-sees[t] // page)]).cuda().long()
        keys, values = (x[pages].transpose(0, 1).reshape(KV, -1, D)[:, :sees[t]] for x in (k, v))
        check(torch, core[t][None], attention(torch, q[t], gate[t], keys, values)[None], t)


FAR = 4_300_003  # keys: more than 2^31 bytes of a head's rows


def far_tolerance():
    """The decodes' 1e-5 and what sums of FAR keys add to it: at most 4 f32 sums of 2^-23 for a tile of 32 keys
    along a span, of which 128 at least share the keys."""
    return REF_REL_L2 + 4 * (FAR / 32 / 128 + 1) * 2.0 ** -23


@pytest.mark.parametrize("own", [False, True])
def test_a_request_of_more_than_2_gib_in_pages(torch_mod, attn, own):
    """Behind a prefix of FAR keys, or of FAR own keys: positions past 2^31 bytes of a head's rows, in a table
    whose entries name the same 64 pages over and over, so that a key's weight counts as often as it comes."""
    torch, page, n_pages = torch_mod, 16, 64
    rng = np.random.default_rng(3)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    pp = FAR // page if not own else 3
    room = -(-FAR // page) + 1 if own else pp + 2
    table = rng.integers(0, n_pages, (1, room))
    lens = np.array([FAR if own else pp * page + 9, pp * page + 2, pp * page - 3])
    rand = lambda *n, **kw: torch.randn(*n, generator=g, device="cuda", **kw)  # noqa: E731
    k, v = (rand(n_pages, KV, page, D, dtype=torch.float16) for _ in range(2))
    q, gate, core = 2 * rand(3, H, D), rand(3, H, D), torch.full((3, H, D), 5.0, device="cuda")
    sc = attn.SharedScratch(3, int(lens.max()) - pp * page, pp * page)
    attn.attn_decode_paged_shared(q, gate, k, v, dev(torch, table), page, dev(torch, lens),
                                  dev(torch, table[0, :pp]), pp, core, sc,
                                  rows=dev(torch, np.zeros(3)))
    for e in range(3):
        n = int(lens[e])
        times = np.repeat(np.bincount(table[0, :n // page], minlength=n_pages)[:, None], page, 1)
        times[table[0, n // page], :n % page] += 1
        times = torch.from_numpy(times.reshape(-1)).cuda().double()
        keys, values = (x.double().transpose(0, 1).reshape(KV, -1, D) for x in (k, v))
        s = torch.matmul(q[e].double().view(KV, GROUP, D), keys.transpose(1, 2).contiguous()) / 16
        w = torch.exp(s - s.amax(-1, keepdim=True)) * times
        ref = (torch.matmul(w / w.sum(-1, keepdim=True), values).view(H, D) *
               torch.sigmoid(gate[e].double()))
        err = ((core[e].double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
        assert err <= far_tolerance(), (e, float(err))


@pytest.mark.parametrize("own", [False, True])
def test_a_request_of_more_than_2_gib_of_rows(torch_mod, attn, own):
    """The same of contiguous caches [2][FAR][256], as the prefix or as one sequence's own keys."""
    torch = torch_mod
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    rand = lambda *n, **kw: torch.randn(*n, generator=g, device="cuda", **kw)  # noqa: E731
    k, v, ks, vs = (rand(KV, n, D, dtype=torch.float16) for n in (FAR, FAR, 33, 33))
    q, gate, core = 2 * rand(2, H, D), rand(2, H, D), torch.full((2, H, D), 5.0, device="cuda")
    far, near = (k, v), (ks, vs)
    prefix, mine = (near, far) if own else (far, near)
    n_prefix, n_mine = prefix[0].shape[1], mine[0].shape[1]
    sc = attn.SharedScratch(2, n_mine, n_prefix)
    attn.attn_decode_ragged_shared(q, gate, mine[0].view(-1), mine[1].view(-1),
                                   dev(torch, [0, 0], torch.int64), dev(torch, [n_mine, 0]),
                                   *prefix, n_prefix, n_prefix, core, sc)
    for e, parts in enumerate(((prefix, mine), (prefix,))):
        x = q[e].double().view(KV, GROUP, D)
        blocks = ((kk[:, i:i + 200_000].double(), vv[:, i:i + 200_000].double())
                  for kk, vv in parts for i in range(0, kk.shape[1], 200_000))
        top = torch.full((KV, GROUP, 1), -float("inf"), dtype=torch.float64, device="cuda")
        all_w, out = torch.zeros_like(top), torch.zeros(KV, GROUP, D, dtype=torch.float64, device="cuda")
        for kk, vv in blocks:
            s = torch.matmul(x, kk.transpose(1, 2).contiguous()) / 16
            new = torch.maximum(top, s.amax(-1, keepdim=True))
            w = torch.exp(s - new)
            all_w = all_w * torch.exp(top - new) + w.sum(-1, keepdim=True)
            out = out * torch.exp(top - new) + torch.matmul(w, vv)
            top = new
        ref = (out / all_w).view(H, D) * torch.sigmoid(gate[e].double())
        err = ((core[e].double() - ref).norm(dim=-1) / ref.norm(dim=-1)).max()
        assert err <= far_tolerance(), (e, float(err))
