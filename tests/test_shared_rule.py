"""CPU tests of what a decode behind a shared prefix launches (no reference counterpart): the host's rule,
through the launchers of oracle/drop_in_capi.hip."""
from __future__ import annotations

import ctypes
import random
import subprocess
import sys

import pytest

from conftest import ROOT

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


# Calls whose cut the kernel chooses and, for a batch of no own keys, gives every workgroup to the prefix:
# nobody chooses the own keys' span, and its word holds what the workspace held.
NO_SPAN = [(8, 32768, 7988), (8, 16384, 4096), (16, 32768, 1024), (24, 8192, 1024)]


@pytest.mark.parametrize("batch,prefix,max_own", NO_SPAN)
def test_calls_that_leave_no_workgroup_for_the_own_keys(O, batch, prefix, max_own):
    r = rule(O, batch, prefix, max_own)
    assert r["chosen"] and r["balanced"] and r["alone_grid"] == r["grid"]


def test_no_own_keys_need_no_span(O):
    """(In a process of its own: a division by the word 0 would end it.)"""
    code = ("from oracle import oracle as O; f = O.drop_in().drop_shared_own_splits; "
            "assert [f(0, 3, w) for w in (0, 1, 512, 2**32 - 1)] == [0] * 4; "
            "assert [f(n, 3, 512) for n in (1, 512, 513, 5000)] == [1, 1, 2, 3]")
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, (res.returncode, res.stderr)
