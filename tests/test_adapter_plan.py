"""The plan of a step's tokens among adapters (host only)."""
import ctypes

import numpy as np
import pytest

from inferllm_b200 import binding as _b
from inferllm_b200.binding import KernelError


def plan(index, ranks):
    sizes, total = (ctypes.c_int * 4)(), ctypes.c_int()
    args = (_b.ints(index), len(index), _b.ints(ranks), len(ranks), sizes, ctypes.byref(total))
    _b.check(_b.lib().illm_adapter_plan(*args, None))
    out = (ctypes.c_int * total.value)()
    _b.check(_b.lib().illm_adapter_plan(*args, out))
    return list(sizes), list(out)


def unpack(index, ranks):
    (T, slots, groups, chunks), out = plan(index, ranks)
    at, fields = 0, {}
    for name, n in (("counts", 4), ("token_adapter", T), ("order", T), ("places", 4 * T), ("slot_begin", slots + 2), ("slot_adapter", slots + 1), ("slot_group", slots + 2),
                    ("groups", groups), ("tile_chunk", -(-T // 256) + 1), ("chunk_tile", chunks), ("chunk_groups", chunks * 4)):
        fields[name] = out[at:at + n]
        at += -(-n // 4) * 4
    assert at == len(out)
    return (T, slots, groups, chunks), fields


@pytest.mark.parametrize("T", [0, 1, 5, 64, 65, 100, 128, 256, 257, 1000])
@pytest.mark.parametrize("count", [1, 3, 70])
def test_every_token_and_every_rank_group_once(T, count):
    rng = np.random.default_rng(T + count)
    ranks = rng.integers(0, 257, count).tolist()
    index = rng.integers(-1, count, T).tolist()
    (_, slots, groups, chunks), f = unpack(index, ranks)
    named = sorted(set(index) - {-1})
    g_of = lambda a: -(-ranks[a] // 16)  # noqa: E731
    assert slots == len(named) and f["slot_adapter"] == named + [-1]
    assert f["counts"] == [slots, groups, chunks, max([g_of(a) for a in named], default=0)]
    assert f["token_adapter"] == index and sorted(f["order"]) == list(range(T))
    assert f["slot_begin"][-1] == T
    for i, a in enumerate(f["slot_adapter"]):
        tokens = f["order"][f["slot_begin"][i]:f["slot_begin"][i + 1]]
        assert tokens == [t for t in range(T) if index[t] == a]
        mine = f["groups"][f["slot_group"][i]:f["slot_group"][i + 1]]
        assert mine == ([a * 16 + g for g in range(g_of(a))] if a >= 0 else [])
    for place, t in enumerate(f["order"]):
        slot = max(i for i in range(slots + 1) if f["slot_begin"][i] <= place < f["slot_begin"][i + 1])
        assert f["places"][4 * place:4 * place + 4] == [t, index[t], f["slot_group"][slot], g_of(index[t]) if index[t] >= 0 else 0]
    if T <= 32 or (T <= 128 and 4 * slots > T):
        assert chunks == 0
        return
    for tile in range(-(-T // 256)):
        mine = range(f["tile_chunk"][tile], f["tile_chunk"][tile + 1])
        assert all(f["chunk_tile"][c] == tile for c in mine)
        got = [g for c in mine for g in f["chunk_groups"][4 * c:4 * c + 4]]
        want = [a * 16 + g for a in sorted(set(index[256 * tile:256 * tile + 256]) - {-1}) for g in range(g_of(a))]
        assert got == want + [-1] * (-len(want) % 4)
    assert f["tile_chunk"][-1] == chunks


def test_refusals():
    for index, ranks in (([0], []), ([2], [8, 8]), ([-2], [8]), ([0], [257]), ([0], [-1])):
        with pytest.raises(KernelError):
            plan(index, ranks)


def test_the_longest_step():
    index = np.full(524280, -1, dtype=np.int32)
    index[-1] = 0
    assert plan(index, [5])[0][0] == 524280
    with pytest.raises(Exception, match="524281"):
        plan(np.full(524281, -1, dtype=np.int32), [5])
