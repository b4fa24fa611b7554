"""How the feed-forward kernels cut sizes up, swept on the host: nothing is left out and nothing overruns its memory."""
import ctypes as C
import random


def plan_ffn(lib, *args):
    out = [C.c_uint32() for _ in range(4)]
    assert lib.tcab_plan_ffn(*args, *[C.byref(o) for o in out]) == 0
    return [o.value for o in out]


def test_every_contraction_is_covered(tcab_lib):
    rng = random.Random(7)
    for _ in range(4000):
        m, n, k = (max(1, int(2 ** rng.uniform(0, 14))), 8 * max(1, int(2 ** rng.uniform(0, 11))), 8 * int(2 ** rng.uniform(0, 11)))
        if rng.random() < 0.05:
            k = 0
        form, pairs, sms = rng.randrange(4), rng.choice([1, 2]), rng.choice([148, 148, 132, 2])
        rows, cols, ranges, blocks = plan_ffn(tcab_lib, form, m, n, k, pairs, sms)
        assert (rows, cols) in {(512, 256), (256, 256), (128, 128), (16, 128), (32, 128), (64, 128)} or \
            (form == 1 and (rows, cols) in {(512, 128), (256, 128), (128, 64), (16, 64), (32, 64), (64, 64)})
        all_blocks = -(-k // 64) * (pairs if form == 2 else 1)
        assert ranges in (1, 2, 4, 8) and ranges * blocks >= all_blocks
        if rows <= 64:  # the receive buffers of a tile cover its rows
            assert m <= rows
        if ranges > 1:  # a CTA of a cluster owns at least eight columns
            assert (64 if form == 1 else 128) // ranges >= 8 and blocks >= 2


def test_one_token_is_cut_over_the_gpu(tcab_lib):
    rows, cols, ranges, blocks = plan_ffn(tcab_lib, 0, 1, 4096, 4096, 1, 148)
    assert rows == 16 and ranges * (4096 // cols) > 100 and ranges * blocks >= 64
    rows, cols, ranges, _ = plan_ffn(tcab_lib, 0, 8192, 8192, 8192, 1, 148)
    assert (rows, cols, ranges) == (512, 256, 1)


def test_layernorm_backward_rings_fit(tcab_lib):
    rng = random.Random(8)
    sizes = [(rows, cols) for cols in list(range(1, 300)) + [511, 512, 513, 1001, 1024, 4096, 4097, 5120, 8192, 8193, 12288, 16384, 16385, 50000]
             for rows in (0, 1, 7, 147, 148, 149, 5000)]
    sizes += [(int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 17))) for _ in range(2000)]
    for rows, cols in sizes:
        for es in (2, 4):
            for aligned in (0, 1):
                out = (C.c_uint32 * 8)()
                assert tcab_lib.tcab_plan_layernorm_backward(rows, cols, es, aligned, 148, out) == 0
                kind, values, tpr, groups, per_group, stages, plane, parts = out
                assert parts >= 1 and parts <= 65535
                if kind == 1:
                    continue
                assert aligned and tpr * groups <= 512 and (tpr * groups) % 32 == 0 and 2 <= stages <= 8
                assert tpr * values >= cols and (tpr in (8, 16, 32) or tpr % 32 == 0)
                # a chunk starts up to 15 bytes behind a 16-byte boundary and is copied to the next one
                assert plane >= groups * per_group * cols * es + 30 and plane % 128 == 0
                assert 2 * plane * stages <= 208 * 1024
                assert groups * cols * 4 <= 2 * plane * stages  # the groups' column sums lie over the ring
                assert groups <= 15 or tpr <= 32  # one named barrier per group of several warps
                assert parts <= 148 and parts <= max(1, -(-rows // (groups * per_group)))
