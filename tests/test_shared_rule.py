"""CPU tests of what a decode behind a shared prefix launches (no reference counterpart): the host's rule,
through the launchers of oracle/drop_in_capi.hip."""
from __future__ import annotations

import ctypes
import random

import pytest

CUS = 256


def rule(O, batch, prefix, max_own, cus=CUS):
    """Row blocks of a workgroup, spans and tiles of a span (as the host cuts them), workgroups of the prefix
    and of the launch, whether the kernel chooses the cut and the own keys' span, and the workgroups of the
    prefix if it finds no own keys."""
    out = (ctypes.c_uint64 * 8)()
    O.drop_in().drop_shared_rule(batch, prefix, max_own, cus, out)
    return dict(zip(("row_blocks", "spans", "span_tiles", "prefix_grid", "grid", "chosen", "balanced",
                     "alone_grid"), out))


def test_spans_cover_the_prefix(O):
    rng = random.Random(3)
    for _ in range(3000):
        batch, prefix = int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 18))
        own = rng.choice([0, int(2 ** rng.uniform(0, 14))])
        r = rule(O, batch, prefix, own, rng.choice([CUS, CUS, 32, 304]))
        tiles = -(-prefix // 32)
        assert (r["spans"] - 1) * r["span_tiles"] < tiles <= r["spans"] * r["span_tiles"]
        groups = -(-(-(-batch // 4)) // r["row_blocks"])
        assert 2 * groups * r["spans"] <= r["prefix_grid"] <= r["grid"]
        assert not r["chosen"] or r["alone_grid"] <= r["grid"]
        if own == 0:
            assert r["grid"] == r["prefix_grid"] and not r["chosen"] and not r["balanced"]


@pytest.mark.parametrize("max_own", [0, 50])
def test_no_prefix(O, max_own):
    r = rule(O, 9, 0, max_own)
    assert r["spans"] == r["prefix_grid"] == 0 and (r["grid"] == 0) == (max_own == 0)
