"""Index arithmetic of a split product, on the CPU: every block of every tile is taken once, no two (CTA, tile) pairs share a record,
all records lie inside the scratch that the host allocates, and the join adds exactly the records that were written."""
import ctypes as C
import random

import pytest


def _lib():
    from iris_testing_b200 import _native
    try:
        lib = _native.lib()
    except Exception as exc:        # no nvcc and no prebuilt library on this machine
        pytest.skip(f"native library unavailable: {exc}")
    lib.b200_linear_record_floats.argtypes = [C.c_int] * 6
    lib.b200_linear_record_floats.restype = C.c_longlong
    return lib


def tile_tokens(mode, M, N, G):
    n = N if mode == 2 else M
    if mode == 2:
        return 64 if n <= 64 else 128 if n <= 128 else 256
    for tt in (16, 32, 64, 128):
        if n <= tt * G:
            return tt
    return 256


def test_records_are_distinct_and_inside_the_scratch():
    lib = _lib()
    rng = random.Random(0)
    for _ in range(400):
        mode, grouped = rng.choice([0, 1, 2]), rng.random() < 0.5
        G = rng.choice([1, 2, 5, 64, 128]) if grouped and mode != 2 else 1
        M, N, K = rng.choice([1, 3, 16, 17, 200, 1000]), 8 * rng.randint(1, 300), 8 * rng.randint(1, 300)
        sms = rng.choice([1, 5, 148])
        tt = tile_tokens(mode, M, N, G)
        if grouped and mode != 2:                       # any sizes that fit, empty groups and rows behind the last among them
            cuts = sorted(rng.randint(0, M) for _ in range(G))
            rows = [b - a for a, b in zip([0] + cuts, cuts)]
        else:
            rows = [N if mode == 2 else M]
        features, depth = (N, K) if mode == 0 else (K, N) if mode == 1 else (K, M)
        tiles = sum(-(-r // tt) for r in rows) * -(-features // 128)
        blocks = -(-depth // 64)
        ctas = (2 if tt <= 64 else 1) * sms
        units = tiles * blocks
        quota = max(4, -(-units // ctas))
        seen, covered = {}, 0
        for cta in range(ctas):
            u, end = min(units, quota * cta), min(units, quota * (cta + 1))
            while u < end:
                t = u // blocks
                n = min(end, (t + 1) * blocks) - u
                assert cta + t not in seen
                seen[cta + t] = t
                covered += n
                u += n
        assert covered == units
        floats = lib.b200_linear_record_floats(mode, M, N, K, G, sms)
        assert not seen or (max(seen) + 1) * 128 * tt <= floats
        for t in range(tiles):
            first, last = t * blocks // quota, ((t + 1) * blocks - 1) // quota
            assert [seen.get(i + t) for i in range(first, last + 1)] == [t] * (last - first + 1)
            assert sum(1 for v in seen.values() if v == t) == last - first + 1 if tiles < 200 else True


def test_rule_never_splits_what_the_kernel_refuses():
    import importlib
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    for M in (1, 16, 17, 300, 5000, 10 ** 6):
        for N, K in ((8, 8), (256, 4096), (28672, 4096), (4096, 14336)):
            for G in (1, 8, 128):
                assert not mod._splits(2, M, N, K, G, True, 148)
                for mode in (0, 1, 2):
                    assert mod._splits(mode, M, N, K, G, False, 148) in (False, True)
    assert mod._splits(0, 1, 28672, 4096, 1, False, 148) and not mod._splits(0, 4096, 4096, 4096, 1, False, 148)
