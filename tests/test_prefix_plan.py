"""The plan of a step's common prefixes, on the host: which tokens walk which positions together."""
import ctypes

import pytest

from inferllm_b200 import binding as _b
from inferllm_b200.binding import KernelError


def plan(groups, lens, G):
    sizes, total = (ctypes.c_int * 7)(), ctypes.c_int()
    args = (len(groups), _b.ints(p for p, _ in groups), _b.ints(len(m) for _, m in groups), _b.ints(t for _, m in groups for t in m), _b.ints(lens), len(lens), G,
            sizes, ctypes.byref(total))
    _b.check(_b.lib().illm_prefix_plan(*args, None))
    out = (ctypes.c_int * max(1, total.value))()
    _b.check(_b.lib().illm_prefix_plan(*args, out))
    flat = list(out)[:total.value]
    tiles = [flat[4 * i:4 * i + 4] for i in range(sizes[0])]
    return dict(tiles=tiles, wide=bool(sizes[1]), longest_prefix=sizes[2], longest_rest=sizes[3], start=flat[sizes[4]:sizes[4] + len(lens)], members=flat[sizes[5]:], per=sizes[6])


def covered(p):
    """token -> positions of the prefix that a tile walks for it."""
    got = {}
    for i, (n, length, *zeros) in enumerate(p["tiles"]):
        assert zeros == [0, 0] and n <= p["per"]
        for t in p["members"][i * p["per"]:i * p["per"] + n]:
            assert t not in got
            got[t] = length
    return got


@pytest.mark.parametrize("G", [1, 3, 4, 7, 16])
@pytest.mark.parametrize("counts", [(1,), (2,), (5, 9), (64,), (300, 17, 1)])
def test_every_member_is_in_one_tile_that_fits(G, counts):
    tokens = sum(counts) + 3
    order = [(i * 7919) % tokens for i in range(tokens)] if tokens % 7919 else list(range(tokens))
    assert sorted(order) == list(range(tokens))
    groups, at = [], 0
    for i, c in enumerate(counts):
        groups.append((64 * (i + 1), order[at:at + c]))
        at += c
    lens = [64 * len(counts) + 1 + t for t in range(tokens)]
    p = plan(groups, lens, G)
    want = {t: length for length, m in groups for t in m}
    assert covered(p) == want
    assert p["start"] == [want.get(t, 0) for t in range(tokens)]
    assert p["per"] == (256 if p["wide"] else 8 if G <= 4 else 16) // G and all(1 <= n for n, *_ in p["tiles"])
    assert p["longest_prefix"] == 64 * len(counts)
    assert p["longest_rest"] == max(n - want.get(t, 0) for t, n in enumerate(lens))


def test_groups_of_many_rows_take_wide_tiles():
    assert not plan([(64, [0, 1])], [65, 65], 16)["wide"]
    assert plan([(64, list(range(64)))], [65] * 64, 4)["wide"]
    for G, most in ((1, 32), (4, 8), (5, 12), (16, 4)):
        assert not plan([(64, list(range(most))), (64, [most + 1])], [65] * (most + 2), G)["wide"] and plan([(64, list(range(most + 1)))], [65] * (most + 1), G)["wide"]


def test_no_groups_is_a_plan():
    p = plan([], [5, 9], 4)
    assert p["tiles"] == [] and p["start"] == [0, 0] and p["longest_rest"] == 9


@pytest.mark.parametrize("groups, lens, G, words", [
    ([(64, [0, 0])], [65, 65], 1, "in two groups"),
    ([(64, [0]), (64, [0])], [65, 65], 1, "in two groups"),
    ([(64, [2])], [65, 65], 1, "outside the step"),
    ([(64, [-1])], [65, 65], 1, "outside the step"),
    ([(64, [])], [65, 65], 1, "at least one token"),
    ([(0, [0])], [65, 65], 1, "at least one position"),
    ([(64, [0, 1])], [65, 63], 1, "fewer than the common prefix"),
    ([], [0], 1, "sees no position"),
    ([], [], 1, "1 to 65535 tokens"),
    ([(64, [0])], [65], 17, "1 to 16 query heads"),
    ([(64, [0])], [65], 0, "1 to 16 query heads"),
])
def test_refusals(groups, lens, G, words):
    with pytest.raises(KernelError, match=words):
        plan(groups, lens, G)


@pytest.mark.parametrize("int8, sequences, positions, kv_heads, once", [
    # as measured, on both sides of the border: bfloat16 rows ...
    (0, 2, 8192, 8, False), (0, 3, 8192, 8, False), (0, 4, 4096, 8, False), (0, 4, 8192, 8, True), (0, 4, 1024, 32, False), (0, 4, 2048, 32, True), (0, 7, 4096, 8, False),
    (0, 8, 2048, 8, False), (0, 8, 4096, 8, True), (0, 16, 2048, 8, False), (0, 16, 4096, 8, True), (0, 32, 1024, 8, False), (0, 32, 2048, 8, True),
    (0, 64, 512, 8, False), (0, 64, 1024, 8, True), (0, 64, 256, 32, True),
    # ... and rows of eight bits
    (1, 2, 4096, 8, False), (1, 2, 8192, 8, True), (1, 4, 256, 32, False), (1, 4, 1024, 32, True), (1, 4, 4096, 8, True), (1, 16, 1024, 8, False), (1, 16, 4096, 8, True),
    (1, 32, 512, 8, False), (1, 32, 2048, 8, True), (1, 64, 512, 8, False), (1, 64, 1024, 8, True),
])
def test_where_common_positions_are_walked_once(int8, sequences, positions, kv_heads, once):
    assert bool(_b.lib().illm_policy_shared_prefix_pays((sequences - 1) * positions * kv_heads, sequences, int8)) == once
