"""The choice of a token per row with settings of its own, against the definition written out in 64 bits (GPU)."""
import numpy as np
import pytest
import torch

from inferllm_b200.kernels import ops

pytestmark = pytest.mark.gpu
INF = float("inf")


def choose(l, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, step by step."""
    l = np.asarray(l, np.float64).copy()
    l[np.isnan(l)] = -INF
    best = l.max()
    if best == -INF:
        return -1
    if not temp > 0:
        return int(np.flatnonzero(l == best)[0])
    with np.errstate(invalid="ignore"):
        w = np.where(l == best, 1.0, np.exp(np.where(l == -INF, -INF, (l - best) / temp)))
    present = int((l > -INF).sum())
    order = np.argsort(-l, kind="stable")[:present]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:int(np.argmax(sums >= max(top_p, 0.0) * sums[-1])) + 1]
    order = order[w[order] >= min(min_p, 1.0)] if min_p > 0 else order
    ids = np.sort(order)
    sums = np.cumsum(w[ids])
    above = sums > u * sums[-1]
    return int(ids[np.argmax(above)]) if above.any() else int(ids[w[ids] > 0][-1])


def f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def check(logits, u, temp, top_k, top_p, min_p):
    got = ops.sample_rows(logits, f32(u), f32(temp), torch.tensor(top_k, dtype=torch.int32, device="cuda"), f32(top_p), f32(min_p)).tolist()
    host, r32 = logits.double().cpu().numpy(), lambda v: float(np.float32(v))
    want = [choose(host[i], r32(u[i]), r32(temp[i]), top_k[i], r32(top_p[i]), r32(min_p[i])) for i in range(len(host))]
    assert got == want


SETTINGS = [(t, k, p, m) for t in (0.0, 0.05, 0.7, 1.0, 3.0) for k in (0, 1, 2, 40, 1500) for p in (1.0, 0.95, 0.3, 0.0) for m in (0.0, 0.05, 1.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 257, 4099, 9001, 32000, 50257, 128256])
def test_settings_of_their_own(V, dtype):
    rng = np.random.default_rng(V)
    rows = [SETTINGS[i] for i in rng.permutation(len(SETTINGS))[:100 if V < 40000 else 40]]
    g = torch.Generator("cuda").manual_seed(V)
    logits = (torch.randn((len(rows), V), generator=g, device="cuda") * 3).to(dtype)
    u = rng.random(len(rows)).astype(np.float32).tolist()
    u[0], u[1 % len(rows)] = 0.0, float(np.float32(1) - np.float32(2) ** -24)
    check(logits, u, *[list(c) for c in zip(*rows)])


def test_rows_of_words_that_cannot_come_and_of_equal_words():
    V = 5000
    n = -3.4028234663852886e38
    rows = torch.zeros((14, V), device="cuda")
    rows[0] = -INF                                  # nothing can come
    rows[1] = float("nan")
    rows[2] = -INF
    rows[2, 4321] = -7.0                            # one word
    rows[3] = n                                     # masked by the type's lowest value: one word is left
    rows[3, 17] = 2.0
    rows[4] = n                                     # all at the lowest value: all alike
    rows[5, 10] = rows[5, 4000] = INF               # infinite words share everything
    rows[6, ::2] = float("nan")                     # every other word, all alike
    rows[7, :] = -0.0                               # the two zeros are alike
    rows[7, ::3] = 0.0
    rows[8] = torch.arange(V, device="cuda") * 1e-3
    rows[9] = -torch.arange(V, device="cuda") * 1e3
    rows[10, :7] = 1e-40                            # subnormal differences
    rows[11] = 1e38
    rows[12] = torch.linspace(-3e38, 3e38, V)
    rows[13, 2500:] = -INF
    for temp, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 100, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 777, 0.9, 0.0), (0.5, 0, 1.0, 0.9), (1e-30, 0, 1.0, 0.0),
                          (1e30, 50, 0.9, 0.1), (0.0, 3, 0.5, 0.5), (1.0, 100000, 0.999, 0.0)):
        for u in (0.0, 0.37, 0.9999):
            check(rows, [u] * 14, [temp] * 14, [k] * 14, [p] * 14, [m] * 14)


def test_few_levels():
    """Words on three levels: cuts fall among equal words, and every border is an exact number."""
    rng = np.random.default_rng(3)
    V, B = 40000, 60
    logits = torch.from_numpy(rng.integers(0, 3, (B, V)).astype(np.float32) * 50).cuda()
    check(logits, rng.random(B).tolist(), [1.0] * B, rng.integers(0, V, B).tolist(), rng.choice([1.0, 0.5, 0.25], B).tolist(), [0.0] * B)


def test_settings_left_out():
    g = torch.Generator("cuda").manual_seed(5)
    logits, u = torch.randn((9, 1234), generator=g, device="cuda"), torch.rand(9, generator=g, device="cuda")
    one, k = torch.ones(9, device="cuda"), torch.zeros(9, dtype=torch.int32, device="cuda")
    want = ops.sample_rows(logits, u, one, k, one, torch.zeros(9, device="cuda")).tolist()
    assert ops.sample_rows(logits, u).tolist() == want
    assert ops.sample_rows(logits, u, one, top_p=one).tolist() == want


def test_rows_apart_and_odd_addresses():
    g = torch.Generator("cuda").manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn((5, 4500), generator=g, device="cuda").to(dtype)
        u, temp = torch.rand(5, generator=g, device="cuda"), torch.full((5,), 0.8, device="cuda")
        for a, b in ((0, 4500), (1, 4400), (3, 4498), (7, 8)):
            part = wide[:, a:b]
            assert ops.sample_rows(part, u, temp).tolist() == ops.sample_rows(part.contiguous(), u, temp).tolist()


def test_a_row_does_not_depend_on_the_batch():
    g = torch.Generator("cuda").manual_seed(7)
    B, V = 200, 32000
    logits, u = torch.randn((B, V), generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    temp, p = torch.rand(B, generator=g, device="cuda") + 0.1, torch.rand(B, generator=g, device="cuda")
    k = torch.randint(0, 300, (B,), generator=g, device="cuda").int()
    whole = ops.sample_rows(logits, u, temp, k, p).tolist()
    for i in range(0, B, 17):
        assert ops.sample_rows(logits[i:i + 1], u[i:i + 1], temp[i:i + 1], k[i:i + 1], p[i:i + 1]).tolist() == whole[i:i + 1]


def test_the_longest_rows():
    g = torch.Generator("cuda").manual_seed(8)
    V = 360448
    logits = torch.randn((3, V), generator=g, device="cuda")
    check(logits, [0.2, 0.6, 0.9], [1.0, 0.8, 0.0], [0, 5000, 3], [0.9, 0.95, 1.0], [0.0, 0.01, 0.0])
    check(torch.zeros((2, V), device="cuda"), [0.2, 0.6], [1.0, 0.8], [0, 5000], [0.9, 1.0], [0.0, 0.01])
    with pytest.raises(ops.KernelError):
        ops.sample_rows(torch.zeros((1, V + 1), device="cuda"), f32([0.5]))


def test_random_numbers_outside_their_range():
    logits = torch.zeros((4, 100), device="cuda")
    assert ops.sample_rows(logits, f32([1.0, 7.0, -1.0, float("nan")])).tolist() == [99, 99, 0, 0]


def test_frequencies():
    """65,536 evenly spaced numbers over one distribution: every word comes as often as its probability says, to one count."""
    B, V = 65536, 50
    l = torch.linspace(-2, 2, V, device="cuda")
    u = (torch.arange(B, device="cuda") + 0.5) / B
    got = torch.bincount(ops.sample_rows(l.expand(B, V).contiguous(), u.float()).long(), minlength=V).double().cpu()
    want = torch.softmax(l.double(), 0).cpu() * B
    assert (got - want).abs().max() <= 1.0


def test_on_another_stream_and_replayed():
    g = torch.Generator("cuda").manual_seed(9)
    logits, u = torch.randn((8, 32000), generator=g, device="cuda"), torch.rand(8, generator=g, device="cuda")
    temp, k = torch.full((8,), 0.9, device="cuda"), torch.full((8,), 50, dtype=torch.int32, device="cuda")
    want = ops.sample_rows(logits, u, temp, k).tolist()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.sample_rows(logits, u, temp, k)
    s.synchronize()
    assert got.tolist() == want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.sample_rows(logits, u, temp, k)
    for seed in range(3):
        logits.copy_(torch.randn((8, 32000), generator=g, device="cuda"))
        graph.replay()
        assert got.tolist() == ops.sample_rows(logits, u, temp, k).tolist()


def test_passes_back_to_back():
    """Many calls with nothing between them, so that their blocks start while others still run."""
    g = torch.Generator("cuda").manual_seed(10)
    cases = []
    for B, V in ((1, 32000), (7, 128256), (64, 32000), (200, 4099), (33, 700)):
        logits, u = torch.randn((B, V), generator=g, device="cuda") * 2, torch.rand(B, generator=g, device="cuda")
        temp, k = torch.rand(B, generator=g, device="cuda") + 0.2, torch.randint(0, 60, (B,), generator=g, device="cuda").int()
        p = torch.rand(B, generator=g, device="cuda") * 0.5 + 0.6
        args = (logits, u, temp, k * (k > 20), p)
        want = ops.sample_rows(*args)
        torch.cuda.synchronize()
        cases.append((args, want))
    got = [ops.sample_rows(*cases[i % 5][0]) for i in range(2000)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, cases[i % 5][1]) for i, t in enumerate(got))


def test_nothing_to_do():
    assert ops.sample_rows(torch.zeros((0, 10), device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)


def test_refusals():
    l, u = torch.zeros((4, 10), device="cuda"), torch.zeros(4, device="cuda")
    bad = [lambda: ops.sample_rows(l.cpu(), u), lambda: ops.sample_rows(l.half(), u), lambda: ops.sample_rows(l[0], u),
           lambda: ops.sample_rows(l.t(), torch.zeros(10, device="cuda")), lambda: ops.sample_rows(l[:, :0], u), lambda: ops.sample_rows(l, u[:3]),
           lambda: ops.sample_rows(l, u.double()), lambda: ops.sample_rows(l, u.cpu()), lambda: ops.sample_rows(l, None),
           lambda: ops.sample_rows(l, u, top_k=u), lambda: ops.sample_rows(l, u, temp=torch.ones(8, device="cuda")[::2]),
           lambda: ops.sample_rows(l[:1].expand(4, 10), u)]
    for call in bad:
        with pytest.raises(ops.KernelError):
            call()


def test_more_words_than_32_bits_count():
    B, V = 17000, 128256
    g = torch.Generator("cuda").manual_seed(9)
    logits = torch.empty((B, V), dtype=torch.bfloat16, device="cuda")
    for r in range(0, B, 1000):
        logits[r:r + 1000] = torch.randn((min(1000, B - r), V), generator=g, device="cuda")
    u, temp = torch.rand(B, generator=g, device="cuda"), torch.full((B,), 0.7, device="cuda")
    top_k = (torch.arange(B, device="cuda") % 3 * 40).int()
    got = ops.sample_rows(logits, u, temp, top_k)
    for r in (0, 2 ** 31 // V - 30, B - 60):
        e = slice(r, r + 60)
        assert torch.equal(got[e], ops.sample_rows(logits[e], u[e].contiguous(), temp[e].contiguous(), top_k[e].contiguous()))


def test_streams_at_once():
    g = torch.Generator("cuda").manual_seed(10)
    logits = torch.randn((24, 40000), generator=g, device="cuda") * 3
    u = torch.rand(24, generator=g, device="cuda")
    top_p = torch.full((24,), 0.9, device="cuda")
    want = ops.sample_rows(logits, u, None, None, top_p)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 3]):
            got.append(ops.sample_rows(logits, u, None, None, top_p))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


@pytest.mark.parametrize("B,V", [(512, 3000), (300, 9000), (513, 3000), (64, 128256)])
def test_more_blocks_than_run_at_once(B, V):
    """Where rows of much work come first, every row still comes, and once: each is what it is in a small batch."""
    g = torch.Generator("cuda").manual_seed(B)
    logits = torch.randn((B, V), generator=g, device="cuda") * 3
    u = torch.rand(B, generator=g, device="cuda")
    kind = torch.randint(0, 5, (B,), generator=g, device="cuda")
    temp = torch.where(kind == 0, 0.0, 0.9)
    top_k = torch.where(kind == 1, 40, torch.where(kind == 2, 700, 0)).int()
    top_p = torch.where((kind == 3) | (kind == 1), 0.8, 1.0)
    out = ops.sample_rows(logits, u, temp, top_k, top_p)
    want = torch.cat([ops.sample_rows(*[v[r:r + 16].contiguous() for v in (logits, u, temp, top_k, top_p)]) for r in range(0, B, 16)])
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(200, 4099), (100, 9001), (16, 32000), (60, 32000), (40, 128256)])
def test_fewer_words_than_top_k_with_top_p(B, V, dtype):
    """Rows of 1 to 39 words that can come, a top_k of 40 and a top_p: the count over the words finds no cut, and a sum of weights
    follows it at once.  On 2, 4 and 8 blocks to a row, few and more of them than run at once, the words all in one block's part
    of the row or in every one, many calls with nothing between them."""
    rng = np.random.default_rng(V + B)
    host = np.full((B, V), -INF)
    for r in range(B):
        n = 1 + r % 39
        at = rng.choice(V, n, replace=False) if r % 3 else (0 if r % 2 else V - 64) + rng.choice(64, n, replace=False)
        host[r, at] = rng.standard_normal(n) * 2
    logits = torch.from_numpy(host.astype(np.float32)).cuda().to(dtype)
    u, top_p = rng.random(B).astype(np.float32).tolist(), [(0.9, 0.5, 0.99)[r % 3] for r in range(B)]
    temp, top_k = [0.8] * B, [40] * B
    check(logits, u, temp, top_k, top_p, [0.0] * B)
    args = logits, f32(u), f32(temp), torch.tensor(top_k, dtype=torch.int32, device="cuda"), f32(top_p)
    want = ops.sample_rows(*args)
    got = [ops.sample_rows(*args) for _ in range(200)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)
