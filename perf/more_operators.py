"""The operators of a batch of requests over a KV page pool, for timing and comparison: the tables and
slots of a step, the preparation of its tokens into pages, and attention behind a prefix that all
requests share.

Kinds:

  plan           page tables, slots and positions from request lengths      attn_page_plan
  prep           norms, rotation and the append to pages                    attn_prep_paged
  shared_paged   decode behind a shared prefix, all keys in pages           attn_decode_paged_shared
  shared_ragged  the same, prefix and own keys in contiguous caches         attn_decode_ragged_shared

Where `own` is false, run() computes them from elementary torch operations in 32 bits (angles in 64);
where it is true, with this package's operators. Shapes are the package's: 16 query heads, 2 KV heads,
head size 256, f16 caches; a page holds [2][page][256] of K or V.
"""
import math

import numpy as np
import torch

own = False

H, KV, D = 16, 2, 256
GROUP = H // KV
SCALE = 1.0 / math.sqrt(D)
STRIDE = 9216  # floats of a token's projections: [16][512] queries and gates, [2][256] k, [2][256] v
EPS = 1e-6
POOL_SPARE = 7  # pages of a pool that no request of a case holds


def listed():
    return [
        # A decode step of 64 chats, one token each; some chats end.
        {"name": "plan_64", "kind": "plan", "batch": 64, "page": 16, "most_len": 4096,
         "most_new": 1, "prefix_pages": 0, "spare_tokens": 0},
        # A busy server's step: prompts of up to 1024 tokens beside decodes, behind a system prompt.
        {"name": "plan_prompts_512", "kind": "plan", "batch": 512, "page": 16, "most_len": 8192,
         "most_new": 1024, "prefix_pages": 64, "spare_tokens": 1000},
        # One chat's next token.
        {"name": "prep_1", "kind": "prep", "n": 1, "seqs": 1, "page": 16, "rope": 64,
         "interleaved": False, "factor": 1.0, "most_pos": 4096, "padding": 0},
        # A decode step of a batch that a graph replays at its largest size: some entries are empty.
        {"name": "prep_64", "kind": "prep", "n": 64, "seqs": 64, "page": 16, "rope": 64,
         "interleaved": False, "factor": 1.0, "most_pos": 262144, "padding": 5},
        # Prompts of an odd total, the whole head rotated in neighbouring pairs, positions scaled.
        {"name": "prep_1001", "kind": "prep", "n": 1001, "seqs": 13, "page": 64, "rope": 256,
         "interleaved": True, "factor": 4.0, "most_pos": 100000, "padding": 0},
        # The engine's chunk.
        {"name": "prep_4096", "kind": "prep", "n": 4096, "seqs": 1, "page": 16, "rope": 64,
         "interleaved": False, "factor": 1.0, "most_pos": 8192, "padding": 0},
        # A few chats behind a short instruction.
        {"name": "shared_3_after_512", "kind": "shared_paged", "batch": 3, "seqs": 3, "page": 16,
         "prefix_pages": 32, "own": 40, "padding": 0},
        # Several questions about one long document.
        {"name": "shared_8_after_32768", "kind": "shared_paged", "batch": 8, "seqs": 8,
         "page": 16, "prefix_pages": 2048, "own": 300, "padding": 0},
        # A server behind one long system prompt, one entry in eight empty.
        {"name": "shared_64_after_32768", "kind": "shared_paged", "batch": 64, "seqs": 64,
         "page": 16, "prefix_pages": 2048, "own": 1024, "padding": 8},
        # Many samples of one prompt.
        {"name": "shared_256_after_8192", "kind": "shared_paged", "batch": 256, "seqs": 256,
         "page": 64, "prefix_pages": 128, "own": 256, "padding": 0},
        # A chunk of one request's prompt: 203 tokens behind 12000, each an entry of its own.
        {"name": "shared_chunk_203_after_12000", "kind": "shared_paged", "batch": 203, "seqs": 1,
         "page": 16, "prefix_pages": 750, "own": 203, "padding": 0},
        # Contiguous caches, a prefix of an odd length, some requests with nothing of their own yet.
        {"name": "shared_ragged_33_after_5003", "kind": "shared_ragged", "batch": 33,
         "prefix": 5003, "own": 900},
    ]


def _log_int(rng, lo, hi):
    """An integer from lo to hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "prep", "shared_paged", "shared_paged", "shared_ragged"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind == "plan":
        batch = _log_int(rng, 1, 512)
        return {"kind": kind, "batch": batch, "page": page, "most_len": _log_int(rng, 1, 16384),
                "most_new": rng.choice([1, 1, _log_int(rng, 2, max(3, 400000 // batch))]),
                "prefix_pages": rng.choice([0, _log_int(rng, 1, 100)]),
                "spare_tokens": rng.choice([0, _log_int(rng, 1, 1000)])}
    if kind == "prep":
        n = _log_int(rng, 1, 4096)
        return {"kind": kind, "n": n, "seqs": _log_int(rng, 1, n), "page": page,
                "rope": rng.choice([8, 32, 64, 64, 128, 256]),
                "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, 2.0, 8.0]),
                "most_pos": _log_int(rng, 1000, 262144),
                "padding": rng.choice([0, _log_int(rng, 1, n + 1) - 1])}
    batch = _log_int(rng, 1, 256)
    prefix = _log_int(rng, 16, min(32768, (1 << 21) // batch))
    own_keys = _log_int(rng, 1, min(1024, 65536 // batch))
    if kind == "shared_ragged":
        return {"kind": kind, "batch": batch, "prefix": prefix, "own": own_keys}
    seqs = rng.choice([batch, batch, _log_int(rng, 1, batch)])
    return {"kind": kind, "batch": batch, "seqs": seqs, "page": page,
            "prefix_pages": max(1, prefix // page), "own": max(own_keys, -(-batch // seqs)),
            "padding": rng.choice([0, _log_int(rng, 1, batch + 1) - 1])}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, dtype=dtype, device="cuda")


def _spread(n, lo, hi, salt=1):
    """n whole numbers of [lo, hi], spread evenly and out of order, the same on every call."""
    i = np.arange(1, n + 1, dtype=np.float64) * salt
    return lo + np.floor((i * 0.6180339887498949) % 1.0 * (hi - lo + 1)).astype(np.int64)


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _plan_sizes(case):
    """Lengths before the step, new tokens, which requests end, and the sizes that follow."""
    b, page, pp = case["batch"], case["page"], case["prefix_pages"]
    behind = _spread(b, 0, case["most_len"], 1)
    fresh = _spread(b, 0, 15, 3) == 0  # places that hold no request yet
    ended = (_spread(b, 0, 15, 5) == 1) & ~fresh
    lens = np.where(fresh, 0, pp * page + np.maximum(behind, 1))
    one = _spread(b, 0, 3, 7) != 0  # most requests decode one token, the others bring a prompt
    new = np.where(one, 1, _spread(b, 1, case["most_new"], 11))
    new[ended] = 0
    held = -(-lens // page)
    room = int(held.max()) + -(-(case["most_new"] + pp * page) // page) + 1
    tokens = int(new.sum()) + case["spare_tokens"]
    return lens, new, ended, held, room, max(tokens, 1)


def _prep_plan(s, g, rng):
    lens, new, ended, held, room, tokens = _plan_sizes(s)
    b, page, pp = s["batch"], s["page"], s["prefix_pages"]
    own_held = np.maximum(held - pp, 0) * (lens > 0)
    grown = np.where(new > 0, -(-(np.where(lens == 0, pp * page, lens) + new) // page), 0)
    wanted = int(np.maximum(grown - np.maximum(held, pp), 0).sum())
    # Mostly enough pages for all; one step in four runs out before its last requests.
    back = int(own_held[ended].sum())
    most = wanted + POOL_SPARE
    free = most if rng.integers(4) else max(wanted - back - 3, 0)
    pool = pp + int(own_held.sum()) + most
    ids = rng.permutation(pool).astype(np.int32)
    prefix, rest, stack = ids[:pp], ids[pp:pool - most], ids[pool - most:][:free]
    table = np.full((b, room), -1, dtype=np.int32)
    first = np.concatenate([[0], np.cumsum(own_held)])
    for r in range(b):
        if lens[r] > 0:
            table[r, :pp] = prefix
            table[r, pp:pp + own_held[r]] = rest[first[r]:first[r + 1]]
    free_pages = np.full(pool, -1, dtype=np.int32)
    free_pages[:free] = stack
    s.update(lens=_dev(lens), new=_dev(new), ended=_dev(ended), table=_dev(table), tokens=tokens,
             prefix=_dev(prefix), free_pages=_dev(free_pages), n_free=_dev(np.array([free])),
             lens_out=torch.zeros(b, dtype=torch.int32, device="cuda"),
             n_free_out=torch.zeros(1, dtype=torch.int32, device="cuda"))


def _frequencies(case):
    """Rotation frequencies: base 1e7 as the engine's model, stretched by `factor` where it is long."""
    i = np.arange(case["rope"] // 2, dtype=np.float64)
    return (1e7 ** (-2.0 * i / case["rope"]) / case["factor"]).astype(np.float32)


def _prep_prep(s, g, rng):
    n, seqs, page = s["n"], min(s["seqs"], s["n"]), s["page"]
    row = np.arange(n) * seqs // n
    start = rng.integers(0, max(1, s["most_pos"] - n), seqs)
    index = np.arange(n) - np.searchsorted(row, np.arange(seqs))[row]  # within the request
    pos = start[row] + index
    block = pos // page - (start // page)[row]  # of the request's pages in this step
    blocks = -(-np.bincount(row, minlength=seqs) // page) + 1  # at most
    pages = int(blocks.sum()) + POOL_SPARE
    ids = rng.permutation(pages)
    slot = ids[np.concatenate([[0], np.cumsum(blocks)])[row] + block] * page + pos % page
    slot[n - s["padding"]:] = -1
    s.update(proj=_randn(g, n, STRIDE), q_norm=1 + 0.2 * _randn(g, D), pages=pages,
             k_norm=1 + 0.2 * _randn(g, D), inv_freq=torch.from_numpy(_frequencies(s)).cuda(),
             rot_scale=1.0 if s["factor"] == 1.0 else 0.1 * math.log(s["factor"]) + 1.0,
             slots=_dev(slot), positions=_dev(pos), q=_randn(g, n, H, D), gate=_randn(g, n, H, D),
             k_pages=_randn(g, pages, KV, page, D, dtype=torch.float16),
             v_pages=_randn(g, pages, KV, page, D, dtype=torch.float16))


def _shared_lens(case):
    """Own keys of every request, and per entry: its request and the own keys it sees."""
    b = case["batch"]
    seqs = min(case.get("seqs", b), b)
    row = np.arange(b) * seqs // b
    count = np.bincount(row, minlength=seqs)
    if case["kind"] == "shared_ragged":
        held = _spread(b, 0, case["own"])
    else:
        held = np.maximum(_spread(seqs, 1, case["own"]), count)
        held[0] = max(case["own"], count[0])
    last = np.cumsum(count)[row] - 1 - np.arange(b)  # entries of the request behind this one
    return held, row, held[row] - last


def _prep_shared(s, g, rng):
    b = s["batch"]
    held, row, sees = _shared_lens(s)
    s.update(q=2.0 * _randn(g, b, H, D), gate=_randn(g, b, H, D),
             core=torch.zeros(b, H, D, device="cuda"), most=int(held.max()))
    if s["kind"] == "shared_ragged":
        total, ctx = int(held.sum()), s["prefix"] + 13
        first = np.concatenate([[0], np.cumsum(held)[:-1]]) * KV * D
        # Where the plain form reads a request's keys, as rows of both heads.
        at = first[:, None, None] // D + np.arange(KV)[:, None] * held[:, None, None]
        at = at + np.minimum(np.arange(max(s["most"], 1)), np.maximum(held[:, None, None] - 1, 0))
        s.update(lens=_dev(held), offsets=_dev(first, torch.int64), prefix_keys=s["prefix"],
                 prefix_ctx=ctx, own_at=_dev(np.minimum(at, max(total * KV - 1, 0)), torch.int64),
                 k=_randn(g, max(total, 1) * KV, D, dtype=torch.float16),
                 v=_randn(g, max(total, 1) * KV, D, dtype=torch.float16),
                 k_prefix=_randn(g, KV, ctx, D, dtype=torch.float16),
                 v_prefix=_randn(g, KV, ctx, D, dtype=torch.float16), sees=_dev(sees))
    else:
        page, pp, seqs = s["page"], s["prefix_pages"], len(held)
        own_pages = -(-held // page)
        pages = pp + int(own_pages.sum()) + POOL_SPARE
        ids = rng.permutation(pages).astype(np.int32)
        table = np.zeros((seqs, pp + int(own_pages.max())), dtype=np.int32)
        first = np.concatenate([[0], np.cumsum(own_pages)]) + pp
        for r in range(seqs):
            table[r, :pp] = ids[:pp]
            table[r, pp:pp + own_pages[r]] = ids[first[r]:first[r + 1]]
        lens = pp * page + sees
        empty = _spread(b, 0, b - 1, 3) < s["padding"]
        lens[empty] = 0
        s.update(lens=_dev(lens), rows=_dev(row) if seqs < b else None, table=_dev(table),
                 prefix_table=_dev(ids[:pp]), prefix_keys=pp * page, of=_dev(row, torch.int64),
                 k=_randn(g, pages, KV, page, D, dtype=torch.float16),
                 v=_randn(g, pages, KV, page, D, dtype=torch.float16))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = dict(case)
    if case["kind"] == "plan":
        _prep_plan(s, g, rng)
    elif case["kind"] == "prep":
        _prep_prep(s, g, rng)
    else:
        _prep_shared(s, g, rng)
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    """What a program holds between its calls."""
    from miso_amd import attention as A

    if s["kind"] == "plan":
        s["plan"] = A.PagePlan(s["batch"], s["tokens"])
    elif s["kind"] != "prep":
        s["scratch"] = A.SharedScratch(s["batch"], s["most"], s["prefix_keys"])


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    from miso_amd import attention as A

    if s["kind"] == "plan":
        p = s["plan"]
        A.attn_page_plan(s["lens"], s["new"], s["table"], s["page"], s["free_pages"], s["n_free"],
                         p, lens_out=s["lens_out"], n_free_out=s["n_free_out"], ended=s["ended"],
                         prefix_table=s["prefix"], prefix_pages=s["prefix_pages"])
        return {"table": s["table"], "free_pages": s["free_pages"], "n_free": s["n_free_out"],
                "lens": s["lens_out"], "status": p.status, "starts": p.starts, "slots": p.slots,
                "positions": p.positions, "rows": p.rows, "visible": p.visible}
    if s["kind"] == "prep":
        proj = s["proj"]
        A.attn_prep_paged(proj, proj.view(-1)[8192:], proj.view(-1)[8704:], s["q_norm"],
                          s["k_norm"], s["inv_freq"], s["k_pages"], s["v_pages"], s["page"],
                          s["slots"], s["positions"], s["q"], s["n"], STRIDE, EPS, gate=s["gate"],
                          rope_dims=s["rope"], interleaved=s["interleaved"],
                          rot_scale=s["rot_scale"])
        return {"q": s["q"], "gate": s["gate"], "k": s["k_pages"], "v": s["v_pages"]}
    if s["kind"] == "shared_paged":
        A.attn_decode_paged_shared(s["q"], s["gate"], s["k"], s["v"], s["table"], s["page"],
                                   s["lens"], s["prefix_table"], s["prefix_pages"], s["core"],
                                   s["scratch"], rows=s["rows"])
    else:
        A.attn_decode_ragged_shared(s["q"], s["gate"], s["k"], s["v"], s["offsets"], s["lens"],
                                    s["k_prefix"], s["v_prefix"], s["prefix"], s["prefix_ctx"],
                                    s["core"], s["scratch"])
    return {"core": s["core"]}


def _pages_of(n, page):
    return torch.div(n + (page - 1), page, rounding_mode="floor")


def _plain_plan(s):
    page, pp, tokens = s["page"], s["prefix_pages"], s["tokens"]
    table, b, room = s["table"], s["batch"], s["table"].shape[1]
    lens, new, ended = s["lens"].long(), s["new"].long(), s["ended"] != 0
    stack, pool, dev = s["free_pages"], s["free_pages"].numel(), table.device
    # Pages of ended requests go on the stack, in the order of request and position.
    j = torch.arange(room, device=dev)
    back = ended[:, None] & (j >= pp) & (j < _pages_of(lens, page)[:, None])
    place = s["n_free"].long() + torch.cumsum(back.view(-1).long(), 0) - 1
    padded = torch.cat([stack, stack.new_zeros(1)])
    padded.scatter_(0, torch.where(back.view(-1), place, pool), table.view(-1))
    stack.copy_(padded[:pool])
    top = s["n_free"].long() + back.sum()
    lens = torch.where(ended, 0, lens)
    fresh = (lens == 0) & (new > 0)
    base = torch.where(fresh, pp * page, lens)
    ends = torch.cumsum(new, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    status = torch.where(new == 0, 0, torch.where(base + new > room * page, 2,
                                                  torch.where(ends > tokens, 3, 0)))
    # (what a fresh request holds already is the prefix)
    need = torch.where((new > 0) & (status == 0),
                       _pages_of(base + new, page) - _pages_of(base, page), 0)
    cum = torch.cumsum(need, 0)
    status = torch.where((need > 0) & (cum > top), 1, status)
    fits = status == 0
    need = torch.where(fits, need, 0)
    grows = fits & (new > 0)
    if pp:
        shared = (grows & fresh)[:, None] & (j < pp)
        table.copy_(torch.where(shared, torch.nn.functional.pad(s["prefix"], (0, room - pp)),
                                table))
    k = j - _pages_of(base, page)[:, None]
    mine = (k >= 0) & (k < need[:, None])
    taken = stack[(top - 1 - ((cum - need)[:, None] + k)).clamp(0, pool - 1)]
    table.copy_(torch.where(mine, taken, table))
    s["n_free_out"].copy_(top - need.sum())
    s["lens_out"].copy_(torch.where(grows, base + new, lens))
    t = torch.arange(tokens, device=dev)
    row = torch.searchsorted(ends, t, right=True).clamp(max=b - 1)
    inside = t < ends[-1]
    good = inside & grows[row]
    pos = torch.where(good, base[row] + t - starts[row], 0)
    slot = table[row, pos // page].long() * page + pos % page
    int32 = torch.int32
    return {"table": table, "free_pages": stack, "n_free": s["n_free_out"],
            "lens": s["lens_out"], "status": status.to(int32), "starts": starts.to(int32),
            "slots": torch.where(good, slot, -1).to(int32), "positions": pos.to(int32),
            "rows": torch.where(inside, row, 0).to(int32),
            "visible": torch.where(good, pos + 1, 0).to(int32)}


def _rotate(s, x):
    """x [n][heads][256] with its first `rope` values rotated."""
    r, half = s["rope"], s["rope"] // 2
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    c = (torch.cos(angle) * s["rot_scale"]).float()[:, None]
    z = (torch.sin(angle) * s["rot_scale"]).float()[:, None]
    if s["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * z, a * z + b * c], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:r]
        turned = torch.cat([a * c - b * z, a * z + b * c], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w


def _plain_prep(s):
    n, page, pages = s["n"], s["page"], s["pages"]
    proj, slots = s["proj"], s["slots"].long()
    good = (slots >= 0)[:, None, None]
    qg = proj[:, :8192].view(n, H, 2, D)
    k = _rotate(s, _norm(proj[:, 8192:8704].view(n, KV, D), s["k_norm"]))
    v = proj[:, 8704:9216].view(n, KV, D)
    s["q"].copy_(torch.where(good, _rotate(s, _norm(qg[:, :, 0], s["q_norm"])), s["q"]))
    s["gate"].copy_(torch.where(good, qg[:, :, 1], s["gate"]))
    # Which token each pool row receives (-1: none), the tokens without a slot behind the last row.
    rows = pages * page
    src = torch.full((rows + 1,), -1, dtype=torch.int64, device="cuda")
    src.scatter_(0, torch.where(slots >= 0, slots, rows), torch.arange(n, device="cuda"))
    src = src[:rows].view(pages, 1, page, 1)
    put = lambda pool, x: pool.copy_(torch.where(  # noqa: E731
        src >= 0, x.half()[src.view(-1).clamp(min=0)].view(pages, page, KV, D).transpose(1, 2),
        pool))
    put(s["k_pages"], k)
    put(s["v_pages"], v)
    return {"q": s["q"], "gate": s["gate"], "k": s["k_pages"], "v": s["v_pages"]}


def _plain_keys(s, x):
    """K ("k") or V ("v") in 32 bits: the prefix [2][prefix][256], and every entry's own keys
    [entries][2][most][256]."""
    if s["kind"] == "shared_ragged":
        prefix = s[x + "_prefix"][:, :s["prefix"]].float()
        return prefix, s[x][s["own_at"]].float()
    pp, page, most = s["prefix_pages"], s["page"], s["most"]
    prefix = s[x][s["prefix_table"].long()].float().transpose(0, 1).reshape(KV, pp * page, D)
    behind = s["table"][:, pp:pp + -(-most // page)].long()
    rows = s[x][behind].transpose(1, 2).reshape(behind.shape[0], KV, -1, D)[:, :, :most]
    return prefix, rows.float()[s["of"]]


def _plain_shared(s):
    b, prefix = s["batch"], s["prefix_keys"]
    (kp, ko), (vp, vo) = _plain_keys(s, "k"), _plain_keys(s, "v")
    lens = s["lens"].long() + (prefix if s["kind"] == "shared_ragged" else 0)
    q = (s["q"] * SCALE).view(b, KV, GROUP, D)
    x = torch.matmul(q.transpose(0, 1).reshape(KV, b * GROUP, D), kp.transpose(1, 2).contiguous())
    x = x.view(KV, b, GROUP, prefix).transpose(0, 1)
    y = torch.matmul(q, ko.transpose(2, 3).contiguous())
    at = torch.arange(prefix + y.shape[-1], device="cuda")
    z = torch.cat([x, y], dim=-1).masked_fill_(at >= lens[:, None, None, None], -math.inf)
    top = z.amax(dim=-1, keepdim=True)
    z = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = z.sum(dim=-1, keepdim=True)
    p, o = z[..., :prefix], z[..., prefix:]
    out = torch.matmul(p.transpose(0, 1).reshape(KV, b * GROUP, prefix), vp)
    out = out.view(KV, b, GROUP, D).transpose(0, 1) + torch.matmul(o.contiguous(), vo)
    out = torch.where(total > 0, out / total, 0.0).reshape(b, H, D)
    s["core"].copy_(out / (1 + torch.exp(-s["gate"])))
    return {"core": s["core"]}


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "plan":
        return _plain_plan(s)
    if s["kind"] == "prep":
        return _plain_prep(s)
    return _plain_shared(s)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "plan":
        lens, new, ended, held, room, tokens = _plan_sizes(case)
        page = case["page"]
        moved = int((-(-new // page)).sum() + held[ended].sum())
        return {"bytes": 4 * (6 * case["batch"] + 4 * tokens + 2 * moved), "flops": 0}
    if case["kind"] == "prep":
        n = case["n"] - case["padding"]
        return {"bytes": n * 4 * (STRIDE + 2 * H * D + KV * D + 2), "flops": 12 * n * (H + KV) * D}
    held, row, sees = _shared_lens(case)
    b = case["batch"]
    prefix = case["prefix"] if case["kind"] == "shared_ragged" else (case["prefix_pages"] *
                                                                     case["page"])
    live = b - case.get("padding", 0)
    return {"bytes": 2 * KV * D * 2 * (prefix + int(held.sum())) + 3 * live * H * D * 4,
            "flops": 4 * H * D * (live * prefix + int(sees.sum()))}


def _exact_plan(s):
    page, pp, tokens = s["page"], s["prefix_pages"], s["tokens"]
    lens, new, ended = (s[x].cpu().numpy().astype(np.int64) for x in ("lens", "new", "ended"))
    table, stack = s["table"].cpu().numpy(), s["free_pages"].cpu().numpy()
    top, b, room = int(s["n_free"]), s["batch"], table.shape[1]
    for r in range(b):
        if ended[r]:
            pages = table[r, pp:-(-lens[r] // page)]
            stack[top:top + len(pages)] = pages
            top += len(pages)
            lens[r] = 0
    starts = np.concatenate([[0], np.cumsum(new)])
    out = {x: np.zeros(tokens, dtype=np.int32) for x in ("positions", "rows", "visible")}
    out["slots"] = np.full(tokens, -1, dtype=np.int32)
    status, left, wanted = np.zeros(b, dtype=np.int32), top, 0
    for r in range(b):
        mine = slice(starts[r], min(starts[r + 1], tokens))
        out["rows"][mine] = r
        if new[r] == 0:
            continue
        base = pp * page if lens[r] == 0 else lens[r]
        need = -(-(base + new[r]) // page) - -(-base // page)
        if base + new[r] > room * page or starts[r + 1] > tokens:
            status[r] = 2 if base + new[r] > room * page else 3
            continue
        wanted += need
        if need and wanted > top:
            status[r] = 1
            continue
        if lens[r] == 0:
            table[r, :pp] = s["prefix"].cpu().numpy()
        at = -(-base // page)
        table[r, at:at + need] = stack[left - need:left][::-1]
        left -= need
        pos = base + np.arange(new[r])
        out["positions"][mine], out["visible"][mine] = pos, pos + 1
        out["slots"][mine] = table[r, pos // page] * page + pos % page
        lens[r] = base + new[r]
    return {"table": table, "free_pages": stack, "n_free": np.array([left], dtype=np.int32),
            "lens": lens.astype(np.int32), "status": status, "starts": starts.astype(np.int32),
            **out}


def _exact_prep(s):
    n, page, r = s["n"], s["page"], s["rope"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    turn = torch.polar(torch.full_like(angle, s["rot_scale"]), angle)[:, None]

    def row(x, w):
        x = x.double()
        x = x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / D + EPS) * w.double()
        if s["interleaved"]:
            pairs = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous())
            x[..., :r] = torch.view_as_real(pairs * turn).reshape(*x.shape[:-1], r)
        else:
            pairs = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
            x[..., :r] = torch.cat([pairs.real, pairs.imag], dim=-1)
        return x

    p = s["proj"]
    q, gate = s["q"].double(), s["gate"].double()
    good = s["slots"] >= 0
    at = s["slots"][good].long()
    q[good] = row(p[:, :8192].reshape(n, H, 512)[..., :D], s["q_norm"])[good]
    gate[good] = p[:, :8192].reshape(n, H, 512)[..., D:].double()[good]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    k[at // page, :, at % page] = row(p[:, 8192:8704].reshape(n, KV, D), s["k_norm"])[good]
    v[at // page, :, at % page] = p[:, 8704:].reshape(n, KV, D).double()[good]
    return {"q": q, "gate": gate, "k": k, "v": v}


def _exact_shared(s):
    b, prefix = s["batch"], s["prefix_keys"]
    ragged = s["kind"] == "shared_ragged"
    held, row, _ = _shared_lens(s)
    lens = s["lens"].cpu().numpy().astype(np.int64) + (prefix if ragged else 0)
    out = torch.zeros(b, H, D, dtype=torch.float64, device="cuda")
    table = None if ragged else s["table"].long()
    offsets = s["offsets"].cpu().numpy() if ragged else None

    def keys(x, head):
        if ragged:
            return s[x + "_prefix"][head, :prefix].double()
        return s[x][s["prefix_table"].long(), head].reshape(-1, D).double()

    def own_keys(x, head, e, n):
        if ragged:
            first = int(offsets[e]) // D + head * int(held[e])
            return s[x][first:first + n].double()
        page, pp = s["page"], s["prefix_pages"]
        pages = table[int(row[e]), pp:pp + -(-n // page)]
        return s[x][pages, head].reshape(-1, D)[:n].double()

    for head in range(KV):
        q = s["q"][:, head * GROUP:(head + 1) * GROUP].double()
        kp, vp = keys("k", head), keys("v", head)
        for e0 in range(0, b, 32):  # the prefix's scores of 32 entries at a time
            x = (q[e0:e0 + 32].reshape(-1, D) @ kp.T / 16.0).view(-1, GROUP, prefix)
            for e in range(e0, min(e0 + 32, b)):
                n = int(lens[e])
                if n == 0:
                    continue
                z, v = x[e - e0][:, :n], vp[:n]
                if n > prefix:
                    z = torch.cat([z, q[e] @ own_keys("k", head, e, n - prefix).T / 16.0], dim=1)
                    v = torch.cat([v, own_keys("v", head, e, n - prefix)])
                gate = s["gate"][e, head * GROUP:(head + 1) * GROUP].double()
                out[e, head * GROUP:(head + 1) * GROUP] = (torch.softmax(z, dim=1) @ v *
                                                           torch.sigmoid(gate))
    return {"core": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(s)
    if case["kind"] == "prep":
        return _exact_prep(s)
    return _exact_shared(s)
