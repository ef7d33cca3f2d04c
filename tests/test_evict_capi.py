"""CPU tests of the bounded cache's entry points: what they refuse on the host (no launch happens
for a refused call), and that their workspaces cover every smaller call."""
from __future__ import annotations

import ctypes
import random

import pytest

EINVAL = 0x4D41
N, P = None, 0x10000  # P: aligned, never dereferenced
FAR = [0x100000000 * (i + 1) for i in range(16)]  # 4 GiB apart: no two caches here overlap


@pytest.fixture(scope="module")
def lib():
    from miso_amd import _lib
    return _lib.load()


def rejected(rc, lib, needle):
    assert rc == EINVAL
    msg = lib.miso_attn_last_error().decode()
    assert needle in msg, msg


@pytest.mark.parametrize("name,tensors", [("miso_attn_decode_weights", 9),
                                          ("miso_attn_decode_weights_fp8", 11)])
def test_decode_weights_refusals(lib, name, tensors):
    fn = getattr(lib, name)
    need = lib.miso_attn_decode_weights_workspace_bytes(5, 4)
    good = [P] * tensors
    for i in range(tensors):
        bad = list(good)
        bad[i] = N
        rejected(fn(*bad, 5, 10, 4, P, need, N), lib, "pointer")
    rejected(fn(*good, 5, 10, 4, N, need, N), lib, "pointer")
    rejected(fn(*good, 5, 10, 4, P + 8, need, N), lib, "pointer")
    rejected(fn(*good, 0, 10, 4, P, need, N), lib, "len must be >= 1")
    rejected(fn(*good, 11, 10, 4, P, 1 << 30, N), lib, "exceeds max_ctx")
    rejected(fn(*good, 5, 10, 0, P, need, N), lib, "n_splits")
    rejected(fn(*good, 5, 10, 4, P, need - 1, N), lib, "workspace smaller")


@pytest.mark.parametrize("name,tensors", [("miso_attn_prefill_weights", 3),
                                          ("miso_attn_prefill_weights_fp8", 4)])
def test_prefill_weights_refusals(lib, name, tensors):
    fn = getattr(lib, name)
    big = 1 << 40
    good = [P] * tensors
    for i in range(tensors):
        bad = list(good)
        bad[i] = N
        rejected(fn(*bad, 0, 3, 10, P, big, N), lib, "pointer")
    rejected(fn(*good, 0, 3, 10, N, big, N), lib, "pointer")
    rejected(fn(*good, 0, 0, 10, P, big, N), lib, "n must be >= 1")
    rejected(fn(*good, 8, 3, 10, P, big, N), lib, "exceeds max_ctx")
    rejected(fn(*good, 0xFFFFFFFF, 3, 10, P, big, N), lib, "exceeds max_ctx")
    rejected(fn(*good, 0, 3, 0x20000001, P, big, N), lib, "2^29")
    rejected(fn(*good, 0, 3, 10, P, 1024, N), lib, "workspace smaller")


def test_prefill_weights_workspace_covers_smaller_calls(lib):
    """The capacity for (max_n, max_rows) is at least that of every smaller chunk over fewer rows."""
    rng = random.Random(3)
    for fp8 in (0, 1):
        for _ in range(60):
            rows = int(2 ** rng.uniform(0, 18))
            n = min(rows, max(1, int(2 ** rng.uniform(0, 14))))
            cap = lib.miso_attn_prefill_weights_workspace_bytes(n, rows, fp8)
            for _ in range(8):
                m = rng.randint(1, n)
                pos0 = rng.randint(0, rows - m)
                assert lib.miso_attn_prefill_weights_workspace_bytes(m, pos0 + m, fp8) <= cap


MIB = 1 << 20


def test_prefill_weights_workspace_is_bounded_over_any_cache(lib):
    """Beside 16 KiB of halves a token (of a piece: 16384 at most, rounded up to 4) there are at most 64
    MiB of sums, or 64 bytes a row, and 4 MiB of scales and statistics, up to the most rows that a cache
    may have; over e4m3 rows the widened K is 1 KiB a row more."""
    for rows in (1 << 16, 1 << 20, (1 << 20) + 1, 3 << 20, 1 << 23, (1 << 24) + 5, 1 << 29):
        for n in (1, 33, 256, 4096, 16384, 1 << 20):
            halves = (min(n, 16384) + 3) * 16384
            got = lib.miso_attn_prefill_weights_workspace_bytes(n, rows, 0)
            assert got <= halves + max(64 * MIB, 64 * (rows + 31)) + 4 * MIB, (rows, n, got / MIB)
            assert lib.miso_attn_prefill_weights_workspace_bytes(n, rows, 1) <= got + 1024 * (rows + 1)


def key_weights_shapes():
    rng = random.Random(5)
    for pos0 in (0, 1, 31, 32, 33, 4000, 4095, 4096, 12001, 262143, 1 << 20):
        for n in (1, 2, 4, 5, 16, 17, 32, 33, 64, 65, 300, 1000, 4096):
            yield pos0, n
    for _ in range(1500):
        rows = int(2 ** rng.uniform(0, rng.choice([13, 19, 24, 29])))
        n = min(rows, max(1, int(2 ** rng.uniform(0, 20))))
        yield rng.choice([0, rows - n, rng.randint(0, rows - n)]), n


def test_prefill_weights_workspace_covers_what_a_launch_uses(lib, O):
    """The capacity holds the chunk's layout, and the layout what each piece's kernels index: the halves
    and scales of its column blocks, the statistics of its spans and groups, and its groups' sums
    (a single group has none)."""
    host = O.drop_in()
    layout, piece = (ctypes.c_uint64 * 6)(), (ctypes.c_uint64 * 7)()
    rng = random.Random(6)
    for pos0, n in key_weights_shapes():
        rows = pos0 + n
        for fp8 in (0, 1):
            host.drop_key_weights_layout(pos0, n, fp8, layout)
            halves, scale, stats, sums, wide, end = layout
            assert all(x % 256 == 0 for x in layout)
            assert end - wide >= (1024 * rows if fp8 else 0)
            more = rng.randint(0, 5000)
            for max_n, max_rows in ((n, rows), (n + more, rows + more), (n, rows + 100 * more)):
                if max_rows <= 1 << 29:
                    cap = lib.miso_attn_prefill_weights_workspace_bytes(max_n, max_rows, fp8)
                    assert cap >= end, (pos0, n, max_n, max_rows)
        host.drop_key_weights_piece(pos0, n, 0, piece)
        most = piece[0]
        count = -(-n // most)
        for i in {0, 1, count // 2, count - 2, count - 1, rng.randrange(count)}:
            if not 0 <= i < count:
                continue
            host.drop_key_weights_piece(pos0, n, i * most, piece)
            m, blocks, waves, groups, row_tiles, spans, span = piece
            at = (pos0, n, i)
            assert m == min(most, n - i * most) and blocks == -(-m // 4), at
            assert groups * waves >= blocks > (groups - 1) * waves and waves in (4, 8), at
            assert 32 * row_tiles >= pos0 + i * most + m > 32 * (row_tiles - 1), at
            assert 0 < spans <= 256 * (8 // waves) and span > 0, at
            assert scale - halves >= 2 * blocks * 32768, at
            assert stats - scale >= 2 * blocks * 4, at
            assert sums - stats >= (spans + 2 * groups) * 32 * waves * 8, at
            assert groups == 1 or wide - sums >= 2 * groups * row_tiles * 32 * 4, at


def test_select_refusals(lib):
    fn = lib.miso_attn_evict_select
    ws = lib.miso_attn_evict_workspace_bytes(100)
    rejected(fn(N, 100, 100, 10, 1, 1, P, P, ws, N), lib, "pointer")
    rejected(fn(P, 100, 100, 10, 1, 1, N, P, ws, N), lib, "pointer")
    rejected(fn(P, 100, 100, 10, 1, 1, P + 2, P, ws, N), lib, "pointer")
    rejected(fn(P, 100, 100, 10, 1, 1, P, N, ws, N), lib, "pointer")
    rejected(fn(P, 101, 100, 10, 1, 1, P, P, ws, N), lib, "exceeds max_ctx")
    rejected(fn(P, 100, 100, 0, 0, 0, P, P, ws, N), lib, "keep")
    rejected(fn(P, 100, 100, 101, 0, 0, P, P, ws, N), lib, "keep")
    rejected(fn(P, 0, 100, 1, 0, 0, P, P, ws, N), lib, "keep")
    rejected(fn(P, 100, 100, 10, 6, 5, P, P, ws, N), lib, "sinks + recent")
    rejected(fn(P, 100, 100, 10, 0xFFFFFFFF, 5, P, P, ws, N), lib, "sinks + recent")
    rejected(fn(P, 0x80000000, 0x80000000, 10, 6, 4, P, P, 1 << 40, N), lib, "2^31")
    rejected(fn(P, 100, 100, 10, 1, 1, P, P, ws - 1, N), lib, "workspace smaller")


def test_select_workspace_covers_smaller_calls(lib):
    sizes = [lib.miso_attn_evict_workspace_bytes(n) for n in
             (0, 1, 2048, 16384, 16385, 17408, 17409, 65536, 65537, 66561, 262144, 1 << 30)]
    assert sizes == sorted(sizes)


def test_gather_refusals(lib):
    fn, fn8 = lib.miso_attn_evict_gather, lib.miso_attn_evict_gather_fp8
    k, v, w, i, ko, vo, wo = FAR[:7]
    for bad in range(7):
        a = [k, v, w, i, ko, vo, wo]
        a[bad] = N
        rejected(fn(a[0], a[1], a[2], 100, a[3], 10, a[4], a[5], a[6], 20, N), lib, "pointer")
    rejected(fn(k, v, w, 100, i, 0, ko, vo, wo, 20, N), lib, "keep must be >= 1")
    rejected(fn(k, v, w, 9, i, 10, ko, vo, wo, 20, N), lib, "exceeds max_ctx")
    rejected(fn(k, v, w, 100, i, 10, ko, vo, wo, 9, N), lib, "exceeds out_ctx")
    # in place, a destination inside the source's last row, and two destinations that share memory
    rejected(fn(k, v, w, 100, i, 10, k, vo, wo, 20, N), lib, "overlaps")
    rejected(fn(k, v, w, 100, i, 10, ko, v + 2 * 100 * 512 - 16, wo, 20, N), lib, "overlaps")
    rejected(fn(k, v, w, 100, i, 10, ko, vo, w, 20, N), lib, "overlaps")
    rejected(fn(k, v, w, 100, i, 10, ko, vo, i + 4, 20, N), lib, "overlaps")
    rejected(fn(k, v, w, 100, i, 10, ko, ko + 512, wo, 20, N), lib, "overlaps")
    k, v, ks, vs, w, i, ko, vo, kso, vso, wo = FAR[:11]
    rejected(fn8(k, v, ks, vs, w, 100, i, 10, ko, vo, kso, vso, wo, 9, N), lib, "exceeds out_ctx")
    rejected(fn8(k, v, ks, vs, w, 100, i, 10, ko, vo, ks, vso, wo, 20, N), lib, "overlaps")
    rejected(fn8(k, v, ks, vs, w, 100, i, 10, ko, vo, kso, kso, wo, 20, N), lib, "overlaps")
    rejected(fn8(k, N, ks, vs, w, 100, i, 10, ko, vo, kso, vso, wo, 20, N), lib, "pointer")


def test_prep_at_refusals(lib):
    for name, n in (("miso_attn_prep_at", 9), ("miso_attn_prep_at_fp8", 11)):
        fn = getattr(lib, name)
        rejected(fn(*[P] * n, 500, 10, 10, 1e-6, N), lib, "KV cache is full")
        rejected(fn(*[N] * n, 500, 1, 10, 1e-6, N), lib, "pointer")
    for name, n in (("miso_attn_prep_batch_at", 9), ("miso_attn_prep_batch_at_fp8", 11)):
        fn = getattr(lib, name)
        rejected(fn(*[P] * n, 500, 8, 10, 1e-6, 3, 9216, N), lib, "KV cache is full")
        rejected(fn(*[P] * n, 0xFFFFFFFE, 0, 10, 1e-6, 3, 9216, N), lib, "2^32")
        rejected(fn(*[P] * n, 500, 0, 10, 1e-6, 3, 9000, N), lib, "proj_stride")
        assert fn(*[N] * n, 500, 0, 10, 1e-6, 0, 9216, N) == 0  # nothing to do


def test_python_refuses_counts_that_do_not_fit():
    from miso_amd import attention as A
    for bad in (-1, 1 << 32):
        with pytest.raises(ValueError):
            A._count(bad, "x")
    with pytest.raises(ValueError):
        A.PrefillWeightsScratch(-1, 10, device="cpu")
    with pytest.raises(ValueError):
        A.EvictScratch(1 << 32, device="cpu")
