"""Page plan and paged prep on the GPU (no reference counterpart): the plan against a plain loop over
requests, the prep against float64."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

H, KV, D, STRIDE = 16, 2, 256, 9216


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def host(t):
    return t.cpu().numpy().astype(np.int64)


def plan_ref(s):
    """One step over the state s (lens, new, ended, table, page, prefix, stack, n_free, tokens, pool)."""
    page, pp, tokens = s["page"], len(s["prefix"]), s["tokens"]
    lens, new, table, stack = (np.array(s[x], dtype=np.int64) for x in
                               ("lens", "new", "table", "stack"))
    b, room = table.shape
    top, cap = int(s["n_free"]), s["table"].shape[1] * page
    for r in range(b):
        if s["ended"][r]:
            back = table[r, pp:min(-(-lens[r] // page), room)].copy()
            stack[top:top + len(back)] = back
            top += len(back)
            lens[r] = 0
    starts = np.concatenate([[0], np.cumsum(new)])
    slots, pos, rows, sees = (np.zeros(tokens, np.int64) for _ in range(4))
    slots[:] = -1
    status, left, wanted = np.zeros(b, np.int64), top, 0
    for r in range(b):
        rows[starts[r]:starts[r + 1]] = r
        if new[r] == 0:
            continue
        base = pp * page if lens[r] == 0 else lens[r]
        if base + new[r] > cap or starts[r + 1] > tokens:
            status[r] = 2 if base + new[r] > cap else 3
            continue
        need = -(-(base + new[r]) // page) - -(-base // page)
        wanted += need
        if need and wanted > top:
            status[r] = 1
            continue
        if lens[r] == 0:
            table[r, :pp] = s["prefix"]
        for j in range(need):
            left -= 1
            table[r, -(-base // page) + j] = stack[left]
        t = np.arange(starts[r], starts[r + 1])
        pos[t] = base + np.arange(new[r])
        g = table[r, pos[t] // page]
        slots[t] = np.where((g >= 0) & (g < s["pool"]), g * page + pos[t] % page, -1)
        sees[t] = pos[t] + 1
        lens[r] = base + new[r]
    return dict(lens=lens, table=table, stack=stack, n_free=left, status=status, starts=starts,
                slots=slots, positions=pos, rows=rows, visible=sees)


def scenario(rng, batch, page, prefix, most_len, most_new, short=False, room=None):
    """Requests of various lengths over a pool in random order."""
    lens = np.where(rng.random(batch) < 0.2, 0, prefix * page + rng.integers(1, most_len + 1, batch))
    new = rng.integers(0, most_new + 1, batch)
    ended = rng.random(batch) < 0.15
    held = -(-lens // page)
    room = room or int(held.max()) + prefix + -(-most_new // page) + 1
    held = np.minimum(held, room)
    own = np.where(lens > 0, np.maximum(held - prefix, 0), 0)
    grown = int((-(-new // page) + 1).sum())
    free = int(rng.integers(0, max(grown // 3, 1))) if short else grown
    pool = prefix + int(own.sum()) + free + 5
    ids = rng.permutation(pool)
    table = np.full((batch, room), -7, np.int64)
    at = prefix
    for r in range(batch):
        if lens[r]:
            table[r, :prefix] = ids[:prefix]
            table[r, prefix:prefix + own[r]] = ids[at:at + own[r]]
            at += own[r]
    stack = np.full(pool, -9, np.int64)
    stack[:free] = ids[at:at + free]
    return dict(lens=lens, new=new, ended=ended, table=table, page=page, prefix=ids[:prefix],
                stack=stack, n_free=free, tokens=max(1, int(new.sum()) + int(rng.integers(0, 9))),
                pool=pool)


def run_plan(torch, attn, s, in_place, with_ended=True):
    d = {x: dev(torch, s[x]) for x in ("lens", "new", "ended", "table", "prefix", "stack")}
    n_free = dev(torch, [s["n_free"]])
    plan = attn.PagePlan(len(s["lens"]), s["tokens"])
    for t in (plan.starts, plan.status, plan.slots, plan.positions, plan.rows, plan.visible):
        t.fill_(-12345)
    out = {} if in_place else dict(lens_out=torch.full_like(d["lens"], -1),
                                   n_free_out=torch.full_like(n_free, -1))
    attn.attn_page_plan(d["lens"], d["new"], d["table"], s["page"], d["stack"], n_free, plan,
                        ended=d["ended"] if with_ended else None, prefix_table=d["prefix"],
                        prefix_pages=len(s["prefix"]), **out)
    if not in_place:
        assert np.array_equal(host(d["lens"]), s["lens"]) and int(n_free) == s["n_free"]
    return dict(lens=host(out.get("lens_out", d["lens"])), table=host(d["table"]),
                stack=host(d["stack"]), n_free=int(out.get("n_free_out", n_free)),
                **{x: host(getattr(plan, x)) for x in ("status", "starts", "slots", "positions",
                                                       "rows", "visible")})


def same(got, want):
    for x in want:
        assert np.array_equal(got[x], want[x]), x


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,prefix,most_len,most_new,short", [
    (1, 8, 0, 1, 1, False), (1, 16, 3, 40, 100, True), (3, 8, 1, 30, 30, False),
    (64, 16, 0, 500, 1, False), (65, 32, 5, 300, 70, True), (257, 16, 2, 100, 50, True),
    (1000, 8, 1, 60, 9, False), (1024, 64, 0, 1000, 1, True), (1025, 8, 2, 40, 5, False),
    (3000, 16, 1, 50, 20, True), (8192, 8, 0, 20, 3, True), (8192, 16, 1, 20, 1, False),
    (5, 65536, 1, 1 << 17, 5000, False), (200, 8, 0, 10, 300, False)])
def test_plan_equals_a_loop(torch_mod, attn, batch, page, prefix, most_len, most_new, short,
                            in_place):
    rng = np.random.default_rng(batch + 7 * page + prefix)
    room = 6 if page == 65536 else None
    s = scenario(rng, batch, page, prefix, most_len, most_new, short, room)
    same(run_plan(torch_mod, attn, s, in_place), plan_ref(s))
    s["ended"] = np.zeros_like(s["ended"])
    same(run_plan(torch_mod, attn, s, in_place, with_ended=False), plan_ref(s))


@pytest.mark.parametrize("batch,prefix,most_len,most_new,short", [
    (300, 70, 1200, 40, False), (300, 70, 1200, 40, True), (2000, 66, 300, 3, True),
    (1500, 130, 90, 30, False), (64, 64, 6000, 1, False), (2, 65, 50000, 9000, False)])
def test_plan_of_many_pages(torch_mod, attn, batch, prefix, most_len, most_new, short):
    """Long prefixes, thousands of pages that go back, prompts of more tokens than one launch places."""
    s = scenario(np.random.default_rng(batch + prefix), batch, 8, prefix, most_len, most_new, short)
    s["ended"][0] = s["lens"][0] > 0
    same(run_plan(torch_mod, attn, s, True), plan_ref(s))


@pytest.mark.parametrize("tokens", [1, 1023, 4096, 4097, 9000])
def test_plan_with_too_few_tokens(torch_mod, attn, tokens):
    """Requests whose tokens end behind max_tokens, by either number of launches."""
    s = scenario(np.random.default_rng(tokens), 700, 8, 2, 90, 40)
    s["tokens"] = tokens
    want = plan_ref(s)
    assert (want["status"] == 3).any() and (tokens == 1 or (want["status"] == 0).any())
    same(run_plan(torch_mod, attn, s, True), want)


def test_plan_refuses_requests_alone(torch_mod, attn):
    """A row too long for its table, tokens behind max_tokens, no pages: the others go on."""
    s = dict(lens=np.array([30, 5, 0, 16, 8, 3]), new=np.array([3, 2, 9, 1, 8, 4]),
             ended=np.zeros(6, bool), page=8, prefix=np.zeros(0, np.int64), pool=40, tokens=25,
             table=np.arange(24).reshape(6, 4), stack=np.concatenate([np.arange(24, 27),
                                                                      np.full(37, -1)]), n_free=3)
    want = plan_ref(s)
    # request 0 needs a fifth page; 2 takes two pages of three, 3 the last, 4 gets none; 5 needs
    # none but its tokens end at 27
    assert want["status"].tolist() == [2, 0, 0, 0, 1, 3]
    same(run_plan(torch_mod, attn, s, True), want)


def test_plan_takes_bad_page_ids_as_no_slot(torch_mod, attn):
    s = dict(lens=np.array([4, 4, 4]), new=np.array([2, 2, 2]), ended=np.zeros(3, bool), page=8,
             prefix=np.zeros(0, np.int64), pool=6, tokens=8, table=np.array([[6], [-1], [5]]),
             stack=np.full(6, 3), n_free=0)
    got = run_plan(torch_mod, attn, s, True)
    same(got, plan_ref(s))
    assert got["slots"].tolist() == [-1, -1, -1, -1, 44, 45, -1, -1]


@pytest.mark.parametrize("pool,refuses", [(900, False), (350, True)])
def test_plan_hands_out_each_page_once(torch_mod, attn, pool, refuses):
    """Steps of a server over one state, updated in place: the pages of the requests, the prefix and the
    stack stay a permutation of the pool, and everything equals the loop. The small pool runs out."""
    rng = np.random.default_rng(5)
    torch, b, page, room, pp = torch_mod, 70, 8, 24, 3
    ids = rng.permutation(pool)
    s = dict(lens=np.zeros(b, np.int64), table=np.full((b, room), -1), page=page, prefix=ids[:pp],
             stack=np.concatenate([ids[pp:], np.full(pp, -1)]), n_free=pool - pp, pool=pool)
    d = {x: dev(torch, s[x]) for x in ("lens", "table", "prefix", "stack")}
    n_free, plan = dev(torch, [s["n_free"]]), attn.PagePlan(b, 700)
    refused = set()
    for step in range(40):
        s["new"] = np.where(rng.random(b) < 0.6, 1, rng.integers(0, 20, b))
        s["ended"] = (rng.random(b) < 0.12) & (s["lens"] > 0)
        s["tokens"] = 700
        attn.attn_page_plan(d["lens"], dev(torch, s["new"]), d["table"], page, d["stack"], n_free,
                            plan, ended=dev(torch, s["ended"]), prefix_table=d["prefix"],
                            prefix_pages=pp)
        want = plan_ref(s)
        got = dict(lens=host(d["lens"]), table=host(d["table"]), stack=host(d["stack"]),
                   n_free=int(n_free), **{x: host(getattr(plan, x)) for x in
                                          ("status", "starts", "slots", "positions", "rows",
                                           "visible")})
        same(got, want)
        refused |= set(want["status"].tolist())
        s.update(lens=want["lens"], table=want["table"], stack=want["stack"],
                 n_free=want["n_free"])
        held = [s["table"][r, pp:-(-s["lens"][r] // page)] for r in range(b)]
        pages = np.concatenate([s["prefix"], s["stack"][:s["n_free"]], *held])
        assert np.array_equal(np.sort(pages), np.arange(pool))
    assert (1 in refused) == refuses


def test_plan_in_a_graph(torch_mod, attn):
    """Steps replayed in place, small and large: each replay is the eager call on the same state."""
    torch = torch_mod
    rng = np.random.default_rng(11)
    for most_new in (1, 600):
        s = scenario(rng, 40, 16, 2, 100, most_new, room=200)
        s["ended"][:] = False
        s["new"] = np.minimum(s["new"], 12) if most_new == 1 else s["new"]
        tokens = s["tokens"]
        state = {x: dev(torch, s[x]) for x in ("lens", "table", "stack")}
        new, prefix = dev(torch, s["new"]), dev(torch, s["prefix"])
        n_free, plan = dev(torch, [s["n_free"]]), attn.PagePlan(40, tokens)

        def call():
            attn.attn_page_plan(state["lens"], new, state["table"], 16, state["stack"], n_free,
                                plan, prefix_table=prefix, prefix_pages=2)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                call()
        torch.cuda.synchronize()
        for step in range(4):
            want = plan_ref(s)
            graph.replay()
            torch.cuda.synchronize()
            same(dict(lens=host(state["lens"]), table=host(state["table"]),
                      stack=host(state["stack"]), n_free=int(n_free),
                      **{x: host(getattr(plan, x)) for x in ("status", "slots", "visible")}),
                 {x: want[x] for x in ("lens", "table", "stack", "n_free", "status", "slots",
                                       "visible")})
            s.update({x: want[x] for x in ("lens", "table", "stack", "n_free")})
            s["new"] = rng.integers(0, 3, 40)
            new.copy_(dev(torch, s["new"]))


# ------------------------------------------------------------------------------------------------
# Prep
# ------------------------------------------------------------------------------------------------

def prep_case(torch, n, page, pages, rope, seed, stride=STRIDE, most_pos=300000):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    return dict(proj=rand(n, stride), q_norm=1 + 0.3 * rand(D), k_norm=1 + 0.3 * rand(D),
                freq=torch.from_numpy((1e4 ** (-2 * np.arange(max(rope // 2, 1)) / max(rope, 1)))
                                      .astype(np.float32)).cuda(),
                k=rand(pages, KV, page, D, dtype=torch.float16),
                v=rand(pages, KV, page, D, dtype=torch.float16),
                slots=dev(torch, rng.permutation(pages * page)[:n]),
                pos=dev(torch, rng.integers(0, most_pos, n)), q=rand(n, H, D), gate=rand(n, H, D))


def run_prep(attn, c, page, rope, interleaved, scale, eps=1e-6, gate=True, **kw):
    n, stride = c["proj"].shape
    flat = c["proj"].view(-1)
    attn.attn_prep_paged(flat, flat[8192:], flat[8704:], c["q_norm"], c["k_norm"], c["freq"], c["k"],
                         c["v"], page, c["slots"], c["pos"], c["q"], n, stride, eps,
                         gate=c["gate"] if gate else None, rope_dims=rope, interleaved=interleaved,
                         rot_scale=scale, **kw)


def prep_ref(torch, c, rope, interleaved, scale, eps=1e-6):
    """(q, k, v, gate) of every token in float64, and q's and k's error bounds: 24 roundings of 2^-24
    (the sum of squares 12, halved, its root 2, two products 2; the f32 angle of up to pi 3.2, sincos
    2, scale 1; two products and their sum 3) of |a| + |b| of the turned pair, scale included."""
    n = c["proj"].shape[0]
    p = c["proj"].double()
    qg = p[:, :8192].reshape(n, H, 2, D)

    def rows(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        tol = x.abs()
        if rope:
            a = c["pos"].double()[:, None, None] * c["freq"].double()[:rope // 2]
            cs, sn = torch.cos(a) * scale, torch.sin(a) * scale
            i = (slice(0, rope, 2), slice(1, rope, 2)) if interleaved else \
                (slice(0, rope // 2), slice(rope // 2, rope))
            u, w_ = x[..., i[0]].clone(), x[..., i[1]].clone()
            x, tol = x.clone(), tol.clone()
            x[..., i[0]], x[..., i[1]] = u * cs - w_ * sn, u * sn + w_ * cs
            tol[..., i[0]] = tol[..., i[1]] = (u.abs() + w_.abs()) * scale
        return x, 24 * 2.0 ** -24 * tol

    return (rows(qg[:, :, 0], c["q_norm"]), rows(p[:, 8192:8704].reshape(n, KV, D), c["k_norm"]),
            p[:, 8704:9216].reshape(n, KV, D), qg[:, :, 1])


def check_prep(torch, c, before, page, ref):
    (q, q_tol), (k, k_tol), v, gate = ref
    slots = c["slots"].long()
    rows = c["k"].shape[0] * page
    good = (slots >= 0) & (slots < rows)
    at = slots[good]
    assert ((c["q"].double() - q).abs() <= q_tol)[good].all()
    assert torch.equal(c["gate"][good], gate.float()[good])
    assert torch.equal(c["q"][~good], before["q"][~good])
    assert torch.equal(c["gate"][~good], before["gate"][~good])
    got = c["k"][at // page, :, at % page].double()
    # half a step of f16 (2^-25 where subnormal) on top
    assert ((got - k[good]).abs() <= k_tol[good] + (k[good].abs() + k_tol[good]) * 2.0 ** -11 +
            2.0 ** -25).all()
    assert torch.equal(c["v"][at // page, :, at % page], v[good].half())
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[at] = False
    for x in "kv":
        flat = c[x].transpose(1, 2).reshape(rows, -1)
        assert torch.equal(flat[untouched], before[x].transpose(1, 2).reshape(rows, -1)[untouched])


@pytest.mark.parametrize("n,page,rope,interleaved,scale", [
    (1, 8, 64, False, 1.0), (1, 16, 64, True, 1.0), (2, 16, 256, False, 1.0), (3, 32, 8, False, 2.0),
    (3, 32, 8, True, 0.5), (5, 16, 0, False, 1.0), (17, 64, 128, True, 1.1386), (64, 16, 64, False, 1.0),
    (65, 8, 24, False, 1.0), (65, 8, 200, True, 1.0), (333, 128, 248, False, 1.3),
    (1001, 16, 256, True, 1.1)])
def test_prep_paged(torch_mod, attn, n, page, rope, interleaved, scale):
    torch = torch_mod
    c = prep_case(torch, n, page, -(-n // page) + 3, rope, n + rope)
    before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
    run_prep(attn, c, page, rope, interleaved, scale)
    check_prep(torch, c, before, page, prep_ref(torch, c, rope, interleaved, scale))


@pytest.mark.parametrize("interleaved", [False, True])
def test_prep_paged_without_a_rotation_takes_no_frequencies(torch_mod, attn, interleaved):
    torch = torch_mod
    c = prep_case(torch, 9, 16, 4, 0, 5)
    c["freq"] = None
    before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
    run_prep(attn, c, 16, 0, interleaved, 1.0)
    check_prep(torch, c, before, 16, prep_ref(torch, c, 0, interleaved, 1.0))
    c["freq"] = torch.zeros(31, device="cuda")
    with pytest.raises(ValueError, match="inv_freq"):
        run_prep(attn, c, 16, 64, interleaved, 1.0)


def test_prep_paged_leaves_tokens_without_a_slot(torch_mod, attn):
    torch = torch_mod
    c = prep_case(torch, 40, 16, 4, 64, 3)
    c["slots"][::3] = -1
    c["slots"][1] = 64
    c["slots"][4] = 2 ** 31 - 1
    c["slots"][7] = -2 ** 31
    c["proj"][::3] = float("nan")
    before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
    run_prep(attn, c, 16, 64, False, 1.0)
    check_prep(torch, c, before, 16, prep_ref(torch, c, 64, False, 1.0))


def test_prep_paged_strides_no_gate_and_far_positions(torch_mod, attn):
    """A wider projection row, no gates, positions to the end of 31 bits, rows of zeros and large
    ones."""
    torch = torch_mod
    c = prep_case(torch, 33, 8, 9, 64, 4, stride=9216 + 20, most_pos=2 ** 31 - 1)
    c["proj"][5] = 0
    c["proj"][6] *= 1e15
    c["proj"][7] *= 1e-15
    before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
    run_prep(attn, c, 8, 64, True, 1.0, gate=False)
    assert torch.equal(c["gate"], before["gate"])
    ref = prep_ref(torch, c, 64, True, 1.0)
    c["gate"] = ref[3].float()
    before["gate"] = c["gate"]
    assert torch.isinf(c["v"][c["slots"][6].long() // 8]).any()  # beyond f16, as the other preps
    check_prep(torch, c, before, 8, ref)


def test_prep_paged_equals_the_contiguous_prep(torch_mod, attn):
    """At small positions the f32 angles of attn_prep_batch are right too: its rows up to roundings."""
    torch, n, page = torch_mod, 50, 16
    c = prep_case(torch, n, page, 4, 64, 9)
    c["slots"] = dev(torch, np.arange(n) + 5)
    c["pos"] = dev(torch, np.arange(n))
    run_prep(attn, c, page, 64, False, 1.0)
    kc, vc = (torch.zeros(KV, n, D, device="cuda", dtype=torch.float16) for _ in range(2))
    q = torch.zeros(n, H, D, device="cuda")
    flat = c["proj"].view(-1)
    attn.attn_prep_batch(flat, flat[8192:], flat[8704:], c["q_norm"], c["k_norm"], c["freq"], kc, vc,
                         q, 0, n, 1e-6, n, STRIDE)
    (_, q_tol), (_, k_tol), _, _ = prep_ref(torch, c, 64, False, 1.0)
    # its angles: pos x inv_freq rounded once more, 50 x 2^-24 at most (a turn by as much)
    assert ((c["q"] - q).abs() <= q_tol * (2 + 50 / 24)).all()
    at = c["slots"].long()
    k = c["k"][at // page, :, at % page].float()
    tol = k_tol * (2 + 50 / 24) + k.abs() * 2.0 ** -10 + 2.0 ** -24
    assert ((k - kc.transpose(0, 1).float()).abs() <= tol).all()
    assert torch.equal(c["v"][at // page, :, at % page], vc.transpose(0, 1))


def test_prep_paged_beyond_4_gib(torch_mod, attn):
    torch, page = torch_mod, 64
    pages = 80000  # 64 KiB each of K and of V: 5.2 GB
    k, v = (torch.empty(pages, KV, page, D, device="cuda", dtype=torch.float16) for _ in range(2))
    c = prep_case(torch, 6, page, 2, 64, 12)
    c["k"], c["v"] = k, v
    c["slots"] = dev(torch, [pages * page - 1, 0, pages * page // 2, 65536 * page, 65536 * page - 1,
                             77])
    mark = {s: (k[s // page, :, s % page].clone()) for s in (1, pages * page - 2)}
    run_prep(attn, c, page, 64, False, 1.0)
    (q, q_tol), (kr, k_tol), vr, _ = prep_ref(torch, c, 64, False, 1.0)
    at = c["slots"].long()
    assert torch.equal(v[at // page, :, at % page], vr.half())
    got = k[at // page, :, at % page].double()
    assert ((got - kr).abs() <= k_tol + kr.abs() * 2.0 ** -10 + 2.0 ** -25).all()
    for s, x in mark.items():
        assert torch.equal(k[s // page, :, s % page].view(torch.int16), x.view(torch.int16))


def test_prep_paged_on_another_stream_and_in_a_graph(torch_mod, attn):
    torch = torch_mod
    c = prep_case(torch, 20, 16, 4, 64, 14)
    c["slots"][17:] = -1
    before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run_prep(attn, c, 16, 64, False, 1.0, stream=side)
    side.synchronize()
    check_prep(torch, c, before, 16, prep_ref(torch, c, 64, False, 1.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_prep(attn, c, 16, 64, False, 1.0)
    for step in range(4):
        c["proj"].normal_()
        c["pos"].random_(0, 100000)
        c["slots"].copy_(dev(torch, np.random.default_rng(step).permutation(70)[:20] - 4))
        before = {x: c[x].clone() for x in ("q", "gate", "k", "v")}
        graph.replay()
        torch.cuda.synchronize()
        check_prep(torch, c, before, 16, prep_ref(torch, c, 64, False, 1.0))
