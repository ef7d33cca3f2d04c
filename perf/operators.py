"""The operators of a bounded KV cache, for timing and comparison: attention that also accumulates
the weight every cached key receives, the choice of the rows to keep by it, and the move of those
rows into another cache.

Kinds:

  decode_weights       one token's gated attention, weights accumulated      attn_decode_weights
  decode_weights_fp8   the same over the e4m3-row cache                      attn_decode_weights_fp8
  prefill_weights      the weights a prompt chunk's tokens give              attn_prefill_weights
  prefill_weights_fp8  the same over the e4m3-row cache                      attn_prefill_weights_fp8
  select               the rows to keep                                      attn_evict_select
  gather               kept rows into another cache                          attn_evict_gather
  gather_fp8           the same over the e4m3-row cache                      attn_evict_gather_fp8

Where `own` is false, run() computes them from elementary torch operations in 32 bits; where it is
true, with this package's operators. Shapes are the package's: 16 query heads, 2 KV heads, head
size 256; caches hold [2][rows][256] f16, or e4m3 codes with one power-of-two scale per row.
"""
import math

import numpy as np
import torch

own = False

H, KV, D = 16, 2, 256
GROUP = H // KV
SCALE = 1.0 / math.sqrt(D)


def listed():
    return [
        # The first tokens of a chat, weights kept from the start: latency is everything.
        {"name": "decode_301", "kind": "decode_weights", "len": 301},
        # One long document, one user.
        {"name": "decode_32768", "kind": "decode_weights", "len": 32768},
        # The largest cache the engine allows.
        {"name": "decode_262144", "kind": "decode_weights", "len": 262144},
        # A long conversation at an odd length, held in 8 bits.
        {"name": "decode_fp8_100003", "kind": "decode_weights_fp8", "len": 100003},
        # The last question of a long prompt votes: a few tokens' weights over all keys.
        {"name": "prefill_33_after_12001", "kind": "prefill_weights", "pos0": 12001, "n": 33},
        # A prompt of ordinary size, every token of it.
        {"name": "prefill_2048", "kind": "prefill_weights", "pos0": 0, "n": 2048},
        # A long prompt's second half.
        {"name": "prefill_8192_after_8192", "kind": "prefill_weights", "pos0": 8192, "n": 8192},
        # A chunk of an odd size in the middle of a prompt, over the 8-bit cache.
        {"name": "prefill_fp8_1001_after_5003", "kind": "prefill_weights_fp8", "pos0": 5003,
         "n": 1001},
        # A short cache, halved.
        {"name": "select_1024_of_2048", "kind": "select", "len": 2048, "keep": 1024, "sinks": 4,
         "recent": 64},
        # The largest cache, cut to a tenth.
        {"name": "select_26215_of_262144", "kind": "select", "len": 262144, "keep": 26215,
         "sinks": 4, "recent": 1024},
        # A quarter of an ordinary cache moves.
        {"name": "gather_8192_of_32768", "kind": "gather", "len": 32768, "keep": 8192},
        # Half of a long 8-bit cache moves, an odd count.
        {"name": "gather_fp8_65535_of_131072", "kind": "gather_fp8", "len": 131072, "keep": 65535},
    ]


def _log_int(rng, lo, hi):
    """An integer from lo to hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode_weights", "decode_weights_fp8", "prefill_weights",
                       "prefill_weights", "prefill_weights_fp8", "select", "gather", "gather_fp8"])
    if kind.startswith("decode"):
        return {"kind": kind, "len": _log_int(rng, 1, 262144)}
    if kind.startswith("prefill"):
        pos0 = rng.choice([0, _log_int(rng, 1, 16000), _log_int(rng, 1024, 16000)])
        n = min(_log_int(rng, 1, 8192), 16384 - pos0)  # never more than the largest listed one
        return {"kind": kind, "pos0": pos0, "n": n}
    if kind == "select":
        n = _log_int(rng, 16, 262144)
        keep = max(1, int(n * rng.uniform(0.02, 0.95)))
        sinks = min(rng.choice([0, 1, 4, 16]), keep)
        recent = min(_log_int(rng, 1, 2048), keep - sinks)
        return {"kind": kind, "len": n, "keep": keep, "sinks": sinks, "recent": recent}
    n = _log_int(rng, 16, 131072)
    return {"kind": kind, "len": n, "keep": max(1, int(n * rng.uniform(0.02, 0.95)))}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, dtype=dtype, device="cuda")


def _fp8_rows(g, rows):
    """Normal rows as e4m3 codes (uint8) and one power-of-two scale per row, the largest code of a
    row in [128, 256)."""
    x = _randn(g, KV, rows, D)
    scale = torch.exp2(torch.floor(torch.log2(x.abs().amax(dim=-1, keepdim=True))) - 7)
    return (x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scale[..., 0].contiguous()


def _some_weights(g, rows, mean):
    """Weights as a run accumulates them: most keys little, a few very much, some none yet."""
    w = torch.exp(1.5 * _randn(g, KV, rows)) * (0.3 * mean)
    return torch.where(torch.rand(KV, rows, generator=g, device="cuda") < 0.05, 0.0, w)


def _out_rows(keep):
    """Rows of the cache that the kept ones move to: room for the next tokens."""
    return keep + 256


def prepare(case, seed):
    kind = case["kind"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if kind.startswith(("decode", "prefill")):
        pos0, n = (case["len"] - 1, 1) if kind.startswith("decode") else (case["pos0"], case["n"])
        rows = pos0 + n
        s.update(pos0=pos0, n=n, rows=rows, q=2.0 * _randn(g, n, H, D),
                 weights=_some_weights(g, rows, 8.0 * n / rows))
        if kind.startswith("decode"):
            s.update(qg=_randn(g, H, 2, D), core=torch.zeros(H, D, device="cuda"))
    else:
        rows = case["len"]
        s.update(rows=rows, weights=_some_weights(g, rows, 1.0))
    if kind.endswith("fp8"):
        s["k"], s["ks"] = _fp8_rows(g, rows)
        s["v"], s["vs"] = _fp8_rows(g, rows)
    elif kind != "select":
        s.update(k=_randn(g, KV, rows, D, dtype=torch.float16),
                 v=_randn(g, KV, rows, D, dtype=torch.float16))
    if kind.startswith("gather"):
        order = torch.rand(KV, rows, generator=g, device="cuda").argsort(dim=1)
        s["index"] = order[:, :case["keep"]].sort(dim=1).values.to(torch.int32).contiguous()
        out = _out_rows(case["keep"])
        s.update(out=out, k_out=torch.zeros(KV, out, D, dtype=s["k"].dtype, device="cuda"),
                 v_out=torch.zeros(KV, out, D, dtype=s["v"].dtype, device="cuda"),
                 weights_out=torch.zeros(KV, out, device="cuda"))
        if kind == "gather_fp8":
            s.update(ks_out=torch.zeros(KV, out, device="cuda"),
                     vs_out=torch.zeros(KV, out, device="cuda"))
    if kind == "select":
        s["index"] = torch.zeros(KV, case["keep"], dtype=torch.int32, device="cuda")
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    """The caches' handles and the scratch that a program holds between its calls."""
    from miso_amd import attention as A

    kind = s["kind"]
    if kind.endswith("fp8"):
        s["cache"] = A.Fp8Cache(0)
        s["cache"].max_ctx = s["rows"]
        s["cache"].k8, s["cache"].v8 = s["k"], s["v"]
        s["cache"].k_scale, s["cache"].v_scale = s["ks"], s["vs"]
    if kind == "gather_fp8":
        s["cache_out"] = A.Fp8Cache(0)
        s["cache_out"].max_ctx = s["out"]
        s["cache_out"].k8, s["cache_out"].v8 = s["k_out"], s["v_out"]
        s["cache_out"].k_scale, s["cache_out"].v_scale = s["ks_out"], s["vs_out"]
    if kind.startswith("decode"):
        s["scratch"] = A.DecodeWeightsScratch(128, s["rows"])
    elif kind == "prefill_weights":
        s["scratch"] = A.PrefillWeightsScratch(s["n"], s["rows"])
    elif kind == "prefill_weights_fp8":
        s["scratch"] = A.PrefillWeightsScratch(s["n"], s["rows"], fp8=True)
    elif kind == "select":
        s["scratch"] = A.EvictScratch(s["len"])


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    from miso_amd import attention as A

    kind = s["kind"]
    if kind == "decode_weights":
        A.attn_decode_weights(s["q"], s["qg"], s["k"], s["v"], s["core"], s["weights"],
                              s["scratch"], s["len"], s["rows"])
        return {"core": s["core"], "weights": s["weights"]}
    if kind == "decode_weights_fp8":
        A.attn_decode_weights_fp8(s["q"], s["qg"], s["cache"], s["core"], s["weights"],
                                  s["scratch"], s["len"])
        return {"core": s["core"], "weights": s["weights"]}
    if kind == "prefill_weights":
        A.attn_prefill_weights(s["q"], s["k"], s["weights"], s["pos0"], s["n"], s["rows"],
                               s["scratch"])
        return {"weights": s["weights"]}
    if kind == "prefill_weights_fp8":
        A.attn_prefill_weights_fp8(s["q"], s["cache"], s["weights"], s["pos0"], s["n"],
                                   s["scratch"])
        return {"weights": s["weights"]}
    if kind == "select":
        A.attn_evict_select(s["weights"], s["len"], s["rows"], s["keep"], s["sinks"], s["recent"],
                            s["index"], s["scratch"])
        return {"index": s["index"]}
    if kind == "gather":
        A.attn_evict_gather(s["k"], s["v"], s["weights"], s["rows"], s["index"], s["keep"],
                            s["k_out"], s["v_out"], s["weights_out"], s["out"])
        return {"k": s["k_out"], "v": s["v_out"], "weights": s["weights_out"]}
    A.attn_evict_gather_fp8(s["cache"], s["weights"], s["index"], s["keep"], s["cache_out"],
                            s["weights_out"])
    return _codes_as_values(s)


def _codes_as_values(s):
    return {"k": s["k_out"].view(torch.float8_e4m3fn), "v": s["v_out"].view(torch.float8_e4m3fn),
            "k_scale": s["ks_out"], "v_scale": s["vs_out"], "weights": s["weights_out"]}


def _plain_rows(s, x):
    """The cache's K ("k") or V ("v") rows in 32 bits."""
    if s["kind"].endswith("fp8"):
        return s[x].view(torch.float8_e4m3fn).float() * s[x + "s"][..., None]
    return s[x].float()


def _plain_attention(s):
    """Softmax weights [2][8 n][rows] of the chunk's queries, row (head of the group, token)."""
    n, rows = s["n"], s["rows"]
    q = s["q"].view(n, KV, GROUP, D).permute(1, 2, 0, 3).reshape(KV, GROUP * n, D) * SCALE
    x = torch.matmul(q, _plain_rows(s, "k").transpose(1, 2).contiguous())
    if n > 1:
        last = s["pos0"] + torch.arange(n, device="cuda").repeat(GROUP)
        x.masked_fill_(torch.arange(rows, device="cuda") > last[:, None], -math.inf)
    x = x.sub_(x.amax(dim=-1, keepdim=True)).exp_()
    return x.div_(x.sum(dim=-1, keepdim=True))


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind.startswith("decode"):
        p = _plain_attention(s)
        o = torch.matmul(p, _plain_rows(s, "v")).view(H, D)
        s["core"].copy_(o / (1 + torch.exp(-s["qg"][:, 1])))
        s["weights"] += p.sum(dim=1)
        return {"core": s["core"], "weights": s["weights"]}
    if kind.startswith("prefill"):
        s["weights"] += _plain_attention(s).sum(dim=1)
        return {"weights": s["weights"]}
    if kind == "select":
        n, sinks, recent = s["len"], s["sinks"], s["recent"]
        middle = s["weights"][:, sinks:n - recent]
        best = middle.sort(dim=1, descending=True, stable=True).indices
        best = best[:, :s["keep"] - sinks - recent] + sinks
        ends = torch.arange(n, device="cuda")
        ends = torch.cat([ends[:sinks], ends[n - recent:]])
        kept = torch.cat([best, ends.expand(KV, -1)], dim=1)
        s["index"].copy_(kept.sort(dim=1).values)
        return {"index": s["index"]}
    keep, at = s["keep"], s["index"].long()
    head = torch.arange(KV, device="cuda")[:, None]
    for name in ("k", "v", "weights") + (("ks", "vs") if kind == "gather_fp8" else ()):
        s[name + "_out"][:, :keep] = s[name][head, at]
    s["weights_out"][:, keep:] = 0
    if kind == "gather_fp8":
        return _codes_as_values(s)
    return {"k": s["k_out"], "v": s["v_out"], "weights": s["weights_out"]}


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    row = D + 4 if kind.endswith("fp8") else 2 * D  # bytes of one K or V row of one KV head
    if kind.startswith("decode"):
        n = case["len"]
        return {"bytes": KV * n * (2 * row + 8) + 4 * H * D * 4, "flops": 4 * H * D * n}
    if kind.startswith("prefill"):
        n, rows = case["n"], case["pos0"] + case["n"]
        pairs = n * case["pos0"] + n * (n + 1) // 2
        return {"bytes": n * H * D * 4 + KV * rows * (row + 8), "flops": 2 * H * D * pairs}
    if kind == "select":
        return {"bytes": 4 * KV * (case["len"] + case["keep"]), "flops": 0}
    keep = case["keep"]
    return {"bytes": KV * (keep * (2 * (2 * row + 4) + 4) + 4 * (_out_rows(keep) - keep)),
            "flops": 0}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "select":
        w = s["weights"].cpu().numpy()
        n, sinks, recent = case["len"], case["sinks"], case["recent"]
        out = []
        for head in w:
            rank = head.astype(np.float64)
            rank[:sinks] = rank[n - recent:] = np.inf  # (an empty slice where recent is 0)
            out.append(np.sort(np.lexsort((np.arange(n), -rank))[:case["keep"]]))
        return {"index": np.stack(out).astype(np.int32)}
    if kind.startswith("gather"):
        keep, out = case["keep"], {}
        names = {"k": "k", "v": "v", "weights": "weights"}
        if kind == "gather_fp8":
            names.update(ks="k_scale", vs="v_scale")
        for name, said in names.items():
            src = s[name]
            if name in ("k", "v") and kind == "gather_fp8":
                src = src.view(torch.float8_e4m3fn).float()
            dst = torch.zeros(KV, s["out"], *src.shape[2:], dtype=torch.float64, device="cuda")
            for head in range(KV):
                dst[head, :keep] = torch.index_select(src[head].double(), 0, s["index"][head])
            out[said] = dst
        return out
    n, pos0, rows = s["n"], s["pos0"], s["rows"]
    weights = s["weights"].double()
    core = torch.zeros(H, D, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 28) // rows)
    key = torch.arange(rows, device="cuda")
    for h in range(H):
        head = h // GROUP
        k = s["k"][head]
        k = (k.view(torch.float8_e4m3fn).float().double() * s["ks"][head].double()[:, None]
             if kind.endswith("fp8") else k.double())
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            x = (s["q"][t0:t1, h].double() @ k.T) / 16.0
            token = torch.arange(t0, t1, device="cuda")
            x = torch.where(key[None, :] <= pos0 + token[:, None], x, -torch.inf)
            p = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
            weights[head] += p.sum(dim=0)
        if kind.startswith("decode"):
            v = s["v"][head]
            v = (v.view(torch.float8_e4m3fn).float().double() * s["vs"][head].double()[:, None]
                 if kind.endswith("fp8") else v.double())
            core[h] = (p[0] @ v) * torch.sigmoid(s["qg"][h, 1].double())
    if kind.startswith("decode"):
        return {"core": core, "weights": weights}
    return {"weights": weights}
