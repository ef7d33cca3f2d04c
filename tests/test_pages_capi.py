"""CPU tests of the entry points for a batch over a page pool: what they refuse on the host (no launch
happens for a refused call), that their workspace covers every smaller call, and the frequencies."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest

EINVAL = 0x4D41
N, P, ODD = None, 0x10000, 0x10002  # P: aligned, never dereferenced


@pytest.fixture(scope="module")
def lib():
    from miso_amd import _lib
    return _lib.load()


def rejected(rc, lib, needle):
    assert rc == EINVAL
    msg = lib.miso_attn_last_error().decode()
    assert needle in msg, msg


PLAN = dict(lens=P, n_new=P, ended=P, page_table=P, batch=3, max_pages=5, page_size=16,
            prefix_table=P, prefix_pages=2, free_pages=P, pool_pages=40, n_free=P, lens_out=P,
            n_free_out=P, status=P, starts=P, slots=P, positions=P, rows=P, visible=P,
            max_tokens=7, stream=N)


@pytest.mark.parametrize("change,needle", [
    *[({x: y}, "4-byte aligned") for y in (N, ODD) for x in PLAN
      if PLAN[x] == P and not (x == "ended" and y is N)],
    ({"batch": 0}, "batch"), ({"batch": 8193}, "batch"),
    ({"page_size": 4}, "power of two"), ({"page_size": 24}, "power of two"),
    ({"page_size": 131072}, "power of two"),
    ({"max_pages": 0}, "max_pages"), ({"max_pages": 1 << 30, "batch": 2}, "max_pages"),
    ({"max_pages": 1 << 27, "batch": 1}, "max_pages"),
    ({"pool_pages": 0}, "pool_pages"), ({"pool_pages": 1 << 27}, "pool_pages"),
    ({"prefix_pages": 6}, "prefix_pages"),
    ({"max_tokens": 0}, "max_tokens"), ({"max_tokens": 1 << 31}, "max_tokens"),
])
def test_page_plan_refusals(lib, change, needle):
    rejected(lib.miso_attn_page_plan(*{**PLAN, **change}.values()), lib, needle)


PREP = dict(qg=P, k=P, v=P, q_norm=P, k_norm=P, inv_freq=P, k_pages=P, v_pages=P, pool_pages=9,
            page_size=16, slots=P, positions=P, q=P, gate=P, n=3, proj_stride=9216, rope_dims=64,
            interleaved=0, rot_scale=1.0, eps=1e-6, stream=N)


@pytest.mark.parametrize("change,needle", [
    *[({x: y}, "aligned") for y in (N, ODD) for x in PREP
      if PREP[x] == P and not (x == "gate" and y is N)],
    ({"pool_pages": 0}, "pool_pages"), ({"pool_pages": 1 << 27}, "pool_pages"),
    ({"page_size": 12}, "power of two"), ({"n": 1 << 31}, "n must be"),
    ({"proj_stride": 9212}, "proj_stride"), ({"proj_stride": 9218}, "proj_stride"),
    ({"rope_dims": 4}, "rope_dims"), ({"rope_dims": 264}, "rope_dims"),
])
def test_prep_paged_refusals(lib, change, needle):
    rejected(lib.miso_attn_prep_paged(*{**PREP, **change}.values()), lib, needle)


def test_prep_paged_of_no_tokens_is_a_no_op(lib):
    assert lib.miso_attn_prep_paged(*{**PREP, "n": 0, "qg": N}.values()) == 0


def shared_paged(lib, **change):
    a = dict(q=P, gate=P, k_pages=P, v_pages=P, page_table=P, max_pages=9, page_size=16, rows=N,
             lens=P, batch=3, max_own=70, prefix_table=P, prefix_pages=4, core=P, workspace=P,
             workspace_bytes=1 << 40, stream=N)
    return lib.miso_attn_decode_paged_shared(*{**a, **change}.values())


@pytest.mark.parametrize("change,needle", [
    *[({x: y}, "aligned") for y in (N, 0x10001) for x in
      ("q", "gate", "k_pages", "v_pages", "page_table", "lens", "prefix_table", "core",
       "workspace")],
    ({"rows": 0x10001}, "aligned"), ({"q": P + 4}, "16-byte"),
    ({"page_size": 7}, "power of two"), ({"max_pages": 0}, "max_pages"),
    ({"max_pages": 1 << 27}, "max_pages"), ({"prefix_pages": 10}, "prefix_pages"),
    ({"max_own": 81}, "max_own"), ({"batch": 0}, "batch"), ({"batch": 65537}, "batch"),
    ({"workspace_bytes": 1000}, "workspace smaller"),
])
def test_decode_paged_shared_refusals(lib, change, needle):
    rejected(shared_paged(lib, **change), lib, needle)


def shared_ragged(lib, **change):
    a = dict(q=P, gate=P, k_cache=P, v_cache=P, kv_offsets=P, lens=P, batch=3, max_own=70,
             k_prefix=P, v_prefix=P, prefix_len=50, prefix_ctx=60, core=P, workspace=P,
             workspace_bytes=1 << 40, stream=N)
    return lib.miso_attn_decode_ragged_shared(*{**a, **change}.values())


@pytest.mark.parametrize("change,needle", [
    *[({x: y}, "aligned") for y in (N, 0x10001) for x in
      ("q", "gate", "k_cache", "v_cache", "kv_offsets", "lens", "k_prefix", "v_prefix", "core",
       "workspace")],
    ({"kv_offsets": P + 4}, "aligned"), ({"prefix_len": 61}, "prefix_ctx"),
    ({"prefix_len": 1 << 31, "prefix_ctx": 1 << 31}, "2^31"), ({"max_own": 1 << 31}, "max_own"),
    ({"batch": 0}, "batch"), ({"batch": 65537}, "batch"),
    ({"workspace_bytes": 1000}, "workspace smaller"),
])
def test_decode_ragged_shared_refusals(lib, change, needle):
    rejected(shared_ragged(lib, **change), lib, needle)


def test_shared_workspace_is_checked_to_the_byte(lib):
    need = lib.miso_attn_decode_shared_workspace_bytes(3, 70, 64)
    rejected(shared_paged(lib, workspace_bytes=need - 1), lib, "workspace smaller")
    need = lib.miso_attn_decode_shared_workspace_bytes(3, 70, 50)
    rejected(shared_ragged(lib, workspace_bytes=need - 1), lib, "workspace smaller")


def test_shared_workspace_covers_smaller_calls(lib):
    need = lib.miso_attn_decode_shared_workspace_bytes
    rng = random.Random(7)
    for _ in range(400):
        b, own, prefix = (int(2 ** rng.uniform(0, x)) for x in (13, 15, 18))
        cap = need(b, own, prefix)
        for _ in range(8):
            assert need(rng.randint(1, b), rng.randint(0, own), rng.randint(0, prefix)) <= cap


def test_wrappers_refuse_host_tensors_and_counts():
    import torch
    from miso_amd import attention as A

    x = torch.zeros(8, dtype=torch.int32)
    plan = A.PagePlan(2, 4, device="cpu")
    with pytest.raises(ValueError, match=r"\[batch\]\[max_pages\]"):
        A.attn_page_plan(x, x, x.view(1, 8), 16, x, x, plan)
    with pytest.raises(ValueError, match="device tensor"):
        A.attn_page_plan(x, x, x.view(2, 4), 16, x, x, plan)
    f, h = torch.zeros(16), torch.zeros(16, dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        A.attn_prep_paged(f, f, f, f, f, f, h, h, 16, x, x, f, 1, 9216, 1e-6)
    with pytest.raises(ValueError, match="2\\^32"):
        A.attn_prep_paged(f, f, f, f, f, f, h, h, 16, x, x, f, -1, 9216, 1e-6)
    sc = A.SharedScratch(4, 10, 64, device="cpu")
    with pytest.raises(ValueError, match="scratch"):
        A.attn_decode_paged_shared(f, f, h, h, x.view(2, 4), 16, torch.zeros(5, dtype=torch.int32),
                                   x, 1, f, sc)
    with pytest.raises(ValueError, match="scratch"):
        A.attn_decode_ragged_shared(f, f, h, h, x, x[:2], h, h, 65, 65, f, sc)
    with pytest.raises(ValueError, match="device tensor"):
        A.attn_decode_ragged_shared(f, f, h, h, x, x[:2], h, h, 5, 5, f, sc)


def test_rope_frequencies():
    from miso_amd import attention as A

    i = np.arange(32)
    plain = 1e7 ** (-2.0 * i / 64)
    got, scale = A.rope_frequencies(64, 1e7, device="cpu")
    assert scale == 1.0 and np.array_equal(got.numpy(), plain.astype(np.float32))
    got, scale = A.rope_frequencies(64, 1e7, factor=4, device="cpu")
    assert scale == 1.0 and np.array_equal(got.numpy(), (plain / 4).astype(np.float32))
    got, scale = A.rope_frequencies(64, 1e4, factor=8, scaling="yarn", original_ctx=4096,
                                    device="cpu")
    base = 1e4 ** (-2.0 * i / 64)
    turns = 4096 * base / (2 * math.pi)
    assert scale == 1 + 0.1 * math.log(8)
    assert np.array_equal(got.numpy()[turns > 32], base[turns > 32].astype(np.float32))
    np.testing.assert_allclose(got.numpy()[turns < 1], base[turns < 1] / 8, rtol=2 ** -23)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (got.numpy()[mid] < base[mid]).all() and (got.numpy()[mid] >
                                                                   base[mid] / 8).all()
    for bad in (dict(rope_dims=12), dict(factor=0.5), dict(scaling="other"), dict(scaling="yarn"),
                dict(base=0.0)):
        with pytest.raises(ValueError):
            A.rope_frequencies(**{"rope_dims": 64, "base": 1e4, "device": "cpu", **bad})
