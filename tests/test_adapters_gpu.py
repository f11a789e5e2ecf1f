"""Low-rank adapters beside a shared projection, against the formula in 64 bits (GPU).

Tolerances.  float32: the K products of a result, and the R behind them, are added in float32, each addition off by at most
2^-24 of a partial sum; partial sums stay within the result's own size, that of one normal variable for the shared product, and
sum |v| |B| for the adapter, so (K + R) 2^-24 times their sum bounds the error.  bfloat16: the result is rounded once, at most
2^-8 of its value; on the prompt path the intermediate values v are rounded as well, which is at most 2^-8 sum |v| |B|.  In the
root-mean-square a rounding to bfloat16 is off by 2^-8 / sqrt(3) times the mean square of where a value lies within its power
of two, 0.0017 of the values; the two of them by 0.0024 of the results, and 2^-8 = 0.0039 is the bound."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from inferllm_b200.kernels import ops

pytestmark = pytest.mark.gpu


def make(T, K, N, ranks, dtype, seed, scale_of=lambda i: 1.0 + 0.5 * i):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    x, w = normal(T, K, std=1.0), normal(N, K, std=K ** -0.5)
    a, b = [normal(r, K, std=K ** -0.5) for r in ranks], [normal(N, r, std=1.0) for r in ranks]
    ad = ops.Adapters(len(ranks), max(max(ranks), 1), N, K, dtype)
    for i, r in enumerate(ranks):
        if r:
            ad.put(i, a[i], b[i], scale_of(i))
    return x, w, a, b, ad, [scale_of(i) for i in range(len(ranks))]


def expected(x, w, a, b, scales, index):
    """(value, |terms| of the adapter) in 64 bits."""
    y, spread = x.double() @ w.double().t(), torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
    index = torch.tensor(index, device="cuda")
    for i in range(len(a)):
        rows = (index == i).nonzero()[:, 0]
        v = scales[i] * (x[rows].double() @ a[i].double().t())
        y[rows] += v @ b[i].double().t()
        spread[rows] = v.abs() @ b[i].double().abs().t()
    return y, spread


def check(got, x, w, a, b, scales, index):
    want, spread = expected(x, w, a, b, scales, index)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    terms = x.shape[1] + max([m.shape[0] for m in a])
    sums = 2.0 ** -24 * terms * (1.0 + want.abs() + spread)
    if x.dtype == torch.float32:
        assert bool((err <= sums).all()), float((err - sums).max())
    else:
        out = 2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0.0
        bound = sums + out + 2.0 ** -8 * spread
        assert bool((err <= bound).all()), float((err - bound).max())
        scale = float((want ** 2).mean().sqrt())
        assert float((err ** 2).mean().sqrt()) <= 2.0 ** -8 * scale


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 8, 16, 17, 33, 64, 65, 127, 130, 256, 257, 300, 600])
def test_tokens(T, dtype):
    ranks = [16, 8, 1, 64, 20, 0, 33]
    rng = np.random.default_rng(T)
    index = rng.integers(-1, len(ranks), T).tolist()
    x, w, a, b, ad, s = make(T, 328, 520, ranks, dtype, T)
    check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(8, 1), (64, 192), (72, 130), (1000, 257), (144, 1001), (4096, 136), (2048, 600)])
def test_sizes(K, N, dtype):
    for T in (1, 9, 40, 100, 290):
        ranks = [4, 16, 48]
        index = [(t * 5) % 4 - 1 for t in range(T)]
        x, w, a, b, ad, s = make(T, K, N, ranks, dtype, K + T)
        check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [1, 7, 16, 17, 64, 65, 128, 200, 256])
def test_ranks(rank, dtype):
    for T in (5, 64, 150):
        x, w, a, b, ad, s = make(T, 256, 264, [rank, 3], dtype, rank + T)
        index = [t % 2 for t in range(T)]
        check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [4, 64, 200, 512])
def test_kinds_of_batches(T, dtype):
    """All with one adapter, none with any, every token with its own, one token with one, prompts one behind another."""
    ranks = [16] * 64
    x, w, a, b, ad, s = make(T, 512, 384, ranks, dtype, 7 * T, lambda i: 0.25 + 0.01 * i)
    for index in ([63] * T, [-1] * T, [t % 64 for t in range(T)], [-1] * (T - 1) + [5], [2] + [-1] * (T - 1), [(t * 4 // T) * 9 - 1 for t in range(T)]):
        check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)


@pytest.mark.parametrize("T,K,N", [(2300, 72, 2304), (2305, 200, 2301), (4097, 64, 1500), (200, 2048, 300), (700, 1104, 520), (5000, 136, 5000)])
def test_large_products(T, K, N):
    """More tiles than pairs of SMs, K in slices; sizes that fill no tile."""
    ranks = [16, 8, 40, 64]
    x, w, a, b, ad, s = make(T, K, N, ranks, torch.bfloat16, T)
    index = [(t // 90) % 5 - 1 for t in range(T)]
    for dtype in (torch.bfloat16, torch.float32):
        check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks), dtype), x, w, a, b, s, index)


def test_no_adapter_is_the_product():
    for T in (3, 64, 100, 500):
        x, w, a, b, ad, s = make(T, 512, 384, [16], torch.float32, T)
        got = ops.linear_adapters(x, w, ad, ops.AdapterRows([-1] * T, ad.ranks))
        assert torch.equal(got, ops.gemm_f32(x, w))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_token_does_not_depend_on_adapters_of_others(dtype):
    """Infinities and NaN in another token's row stay there, and so does an adapter whose values overflow; one that is not
    finite itself is refused."""
    for T in (6, 64, 200, 300):
        x, w, a, b, ad, s = make(T, 320, 272, [16, 32, 8], dtype, T)
        index = [(t * 7) % 4 - 1 for t in range(T)]
        rows = ops.AdapterRows(index, ad.ranks)
        want = ops.linear_adapters(x, w, ad, rows)
        a[1][0] = 3e38
        ad.put(1, a[1], b[1], s[1])
        bad = [t for t in range(T) if index[t] == 1]
        clean = next(t for t in range(T) if index[t] == 0)
        x[clean] = float("nan")
        got = ops.linear_adapters(x, w, ad, rows)
        ok = [t for t in range(T) if index[t] != 1 and t != clean]
        assert torch.equal(got[ok], want[ok])
        assert not torch.isfinite(got[bad]).all() and got[clean].isnan().all()


def test_float32_rows_do_not_depend_on_the_batch():
    T = 70
    x, w, a, b, ad, s = make(T, 500, 300, [16, 24, 5], torch.float32, 1)
    index = [(t * 5) % 4 - 1 for t in range(T)]
    whole = ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks))
    for t in (0, 1, 2, 3, 33, 69):
        one = ops.linear_adapters(x[t:t + 1].contiguous(), w, ad, ops.AdapterRows(index[t:t + 1], ad.ranks))
        assert torch.equal(one[0], whole[t])


@pytest.mark.parametrize("dtype", DTYPES)
def test_put_replaces_and_remove_removes(dtype):
    x, w, a, b, ad, s = make(40, 256, 200, [32, 16], dtype, 3)
    index = [t % 2 for t in range(40)]
    rows = ops.AdapterRows(index, ad.ranks)
    ad.put(0, a[1], b[1], 2.0)                          # a smaller rank: the plan still covers it
    check(ops.linear_adapters(x, w, ad, rows), x, w, [a[1], a[1]], [b[1], b[1]], [2.0, s[1]], index)
    ad.remove(1)
    check(ops.linear_adapters(x, w, ad, rows), x, w, [a[1], a[1]], [b[1], b[1]], [2.0, 0.0], index)
    ad.put(1, a[0], b[0], 1.0)                          # a larger one: it does not
    with pytest.raises(ops.KernelError):
        ops.linear_adapters(x, w, ad, rows)


def test_float32_results_of_bfloat16():
    for T in (3, 64, 100, 300):
        x, w, a, b, ad, s = make(T, 256, 200, [16, 40], torch.bfloat16, T)
        index = [t % 3 - 1 for t in range(T)]
        got = ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks), torch.float32)
        assert got.dtype == torch.float32
        check(got, x, w, a, b, s, index)


@pytest.mark.parametrize("T", [5, 64, 300])
def test_streams_and_graphs(T):
    x, w, a, b, ad, s = make(T, 512, 384, [16, 32], torch.bfloat16, T)
    rows = ops.AdapterRows([t % 3 - 1 for t in range(T)], ad.ranks)
    want = ops.linear_adapters(x, w, ad, rows)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.linear_adapters(x, w, ad, rows)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_adapters(x, w, ad, rows)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").bfloat16())
        graph.replay()
        assert torch.equal(got, ops.linear_adapters(x, w, ad, rows))


def test_calls_back_to_back():
    """Many calls with nothing between them but the kernel that makes their input: what each waits for, it waits for."""
    cases = []
    for T, K, N, dtype in ((1, 512, 600, torch.bfloat16), (20, 1024, 520, torch.bfloat16), (100, 512, 384, torch.bfloat16), (200, 2048, 512, torch.bfloat16),
                           (600, 512, 2304, torch.bfloat16), (2500, 128, 2304, torch.bfloat16), (30, 300, 200, torch.float32)):
        x, w, a, b, ad, s = make(T, K, N, [16, 40, 8], dtype, T + K)
        rows = ops.AdapterRows([(t // 3) % 4 - 1 for t in range(T)], ad.ranks)
        cases.append((x, w, ad, rows, [ops.linear_adapters(x * f, w, ad, rows) for f in (1.0, 2.0)]))
    torch.cuda.synchronize()
    got = []
    for i in range(700):
        x, w, ad, rows, want = cases[i % 7]
        f = i // 7 % 2
        got.append((ops.linear_adapters(x * (1.0 + f), w, ad, rows), want[f]))
        if i % 140 == 139:
            torch.cuda.synchronize()
            assert all(torch.equal(g, v) for g, v in got)
            got = []


def test_refusals():
    x, w, a, b, ad, s = make(4, 64, 32, [8, 8], torch.bfloat16, 1)
    rows = ops.AdapterRows([0, 1, -1, 0], ad.ranks)
    other = ops.Adapters(2, 8, 32, 64, torch.float32)
    bad = [lambda: ops.linear_adapters(x[:3].contiguous(), w, ad, rows), lambda: ops.linear_adapters(x, w[:, :56].contiguous(), ad, rows),
           lambda: ops.linear_adapters(x, w[:16].contiguous(), ad, rows), lambda: ops.linear_adapters(x, w, other, rows),
           lambda: ops.linear_adapters(x.float(), w, ad, rows), lambda: ops.linear_adapters(x.cpu(), w, ad, rows),
           lambda: ops.linear_adapters(x.t().contiguous().t(), w, ad, rows), lambda: ops.linear_adapters(x, w, ad, rows, torch.float16),
           lambda: ops.linear_adapters(x.float(), w.float(), other, rows, torch.bfloat16),
           lambda: ops.linear_adapters(x, w, ad, ops.AdapterRows([0, 2, -1, 0], [8, 8, 8])),
           lambda: ops.linear_adapters(x, w, ad, ops.AdapterRows([0, 1, -1, 0], [8, 0])),
           lambda: ad.put(2, a[0], b[0]), lambda: ad.put(0, a[0][:, :32], b[0]), lambda: ad.put(0, a[0], b[0][:, :4]),
           lambda: ad.put(0, torch.zeros(9, 64), torch.zeros(32, 9)), lambda: ad.put(0, a[0].int(), b[0]),
           lambda: ad.put(0, a[0] * float("inf"), b[0]), lambda: ad.put(0, a[0], b[0] * float("nan")), lambda: ad.put(0, a[0], b[0], float("inf")),
           lambda: ad.put(0, a[0].double() * 1e39, b[0]),
           lambda: ops.Adapters(0, 8, 32, 64), lambda: ops.Adapters(2, 257, 32, 64), lambda: ops.Adapters(2, 8, 32, 60),
           lambda: ops.Adapters(2, 8, 32, 64, torch.float16), lambda: ops.Adapters(2, 8, 32, 64, device="cpu"),
           lambda: ops.AdapterRows([0, 2], [8, 8]), lambda: ops.AdapterRows([-2], [8]), lambda: ops.AdapterRows([0], [300])]
    for call in bad:
        with pytest.raises(ops.KernelError):
            call()


def test_put_takes_parameters_and_its_own_factors():
    x, w, a, b, ad, s = make(6, 64, 48, [16, 8], torch.bfloat16, 3)
    rows = ops.AdapterRows([0, 1, -1, 0, 1, 1], ad.ranks)
    want = ops.linear_adapters(x, w, ad, rows)
    ad.put(0, torch.nn.Parameter(a[0].clone()), torch.nn.Parameter(b[0].clone()), s[0])
    assert not (ad.a.requires_grad or ad.b.requires_grad)
    assert torch.equal(ops.linear_adapters(x, w, ad, rows), want)
    ad.put(0, ad.a[0], ad.b[0, 0], s[0])
    ad.put(1, ad.a[1, :8], ad.b[1, 0, :, :8], s[1])
    assert torch.equal(ops.linear_adapters(x, w, ad, rows), want)
    with pytest.raises(ops.KernelError, match="not finite"):
        ad.put(0, a[0], b[0], 1e39)                     # (no float32)
    assert torch.equal(ops.linear_adapters(x, w, ad, rows), want)


@pytest.mark.parametrize("T", [7, 100, 400])
def test_two_streams_at_once(T):
    x, w, a, b, ad, s = make(T, 512, 1000, [16, 40, 8], torch.bfloat16, T)
    rows = ops.AdapterRows([t % 4 - 1 for t in range(T)], ad.ranks)
    xs = [x, x * 2.0, x * -1.0]
    want = [ops.linear_adapters(v, w, ad, rows) for v in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for i in range(40):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[j].append(ops.linear_adapters(xs[j], w, ad, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[j]) for j in range(3) for g in got[j])


@pytest.mark.parametrize("dtype,N", [(torch.bfloat16, 16400), (torch.bfloat16, 16401), (torch.float32, 16400)])
def test_more_results_than_32_bits_count(dtype, N):
    T, K = 140000, 32
    x, w, a, b, ad, s = make(T, K, N, [8, 24], dtype, N)
    index = [(t // 1000) % 3 - 1 for t in range(T)]
    out = ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks))
    for t in (0, 2 ** 31 // N - 100, T - 200):
        check(out[t:t + 200], x[t:t + 200], w, a, b, s, index[t:t + 200])


def test_captured_first_of_all():
    """A process whose first call is a captured one."""
    code = """
import torch
from inferllm_b200.kernels import ops
x, w = torch.randn(5, 64, device="cuda").bfloat16(), torch.randn(40, 64, device="cuda").bfloat16()
ad = ops.Adapters(1, 8, 40, 64)
ad.put(0, torch.randn(8, 64), torch.randn(40, 8))
rows = ops.AdapterRows([0, -1, 0, 0, -1], ad.ranks)
u = torch.rand(5, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.linear_adapters(x, w, ad, rows, torch.float32)
    ids = ops.sample_rows(y, u)
g.replay()
assert torch.equal(y, ops.linear_adapters(x, w, ad, rows, torch.float32)) and torch.equal(ids, ops.sample_rows(y, u))
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("T", [65, 70, 100, 128])
def test_from_65_to_128_tokens(T):
    """Few adapters (tiles of tokens), many (token by token), and the two on either side of the rule."""
    ranks = [16] * 64
    x, w, a, b, ad, s = make(T, 512, 388, ranks, torch.bfloat16, 5 * T, lambda i: 0.25 + 0.01 * i)
    for used in (1, 2, T // 4, T // 4 + 1, 64):
        for index in ([t % used for t in range(T)], [(t * used // T) if t % 9 else -1 for t in range(T)]):
            check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)
    rows = ops.AdapterRows([t % 3 - 1 for t in range(T)], ad.ranks)
    want = ops.linear_adapters(x, w, ad, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_adapters(x, w, ad, rows)
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("T", [33, 48, 64])
def test_wide_products_of_33_to_64_tokens(T):
    ranks = [16, 64, 40, 8] + [16] * 20
    x, w, a, b, ad, s = make(T, 128, 9600, ranks, torch.bfloat16, 3 * T, lambda i: 0.25 + 0.05 * i)
    for used in (1, 4, T // 4, T // 4 + 1):
        index = [t % used if t % 7 else -1 for t in range(T)]
        check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)


@pytest.mark.parametrize("K,N", [(2752, 160), (1000, 2049), (2048, 4096), (260, 9000), (72, 130), (514, 300)])
def test_float32_rows_by_any_kernel(K, N):
    """A row's bits are the same in products of any number of rows, whichever kernel they take, and an infinite row stays alone."""
    x, w, a, b, ad, s = make(200, K, N, [16, 5], torch.float32, K + N)
    x[7, 3] = float("inf")
    none = [ops.linear_adapters(x[t:t + 8].clone(), w, ad, ops.AdapterRows([-1] * len(x[t:t + 8]), ad.ranks)) for t in range(0, 200, 8)]
    want = torch.cat(none)
    for T in (9, 16, 17, 32, 33, 64, 65, 96, 128, 161, 200):
        got = ops.linear_adapters(x[:T].clone(), w, ad, ops.AdapterRows([-1] * T, ad.ranks))
        same = (got == want[:T]) | (got.isnan() & want[:T].isnan())
        assert bool(same.all()), T
        assert torch.isfinite(got[:7]).all()


@pytest.mark.parametrize("T,K,N", [(200, 4096, 6144), (512, 4096, 4096), (257, 1024, 1024), (1000, 4096, 6144), (2048, 1024, 1024), (2048, 4096, 4096),
                                   (1024, 8192, 1024), (70, 11008, 4096), (200, 4096, 6143), (500, 4096, 4093), (257, 1024, 1021), (1000, 2048, 6139),
                                   (1024, 8192, 1019)])
def test_widths_of_tiles(T, K, N):
    """Sizes for which the estimate takes tiles of every width, some with K in slices; outputs that fill no tile."""
    ranks = [16, 40, 8]
    x, w, a, b, ad, s = make(T, K, N, ranks, torch.bfloat16, T + N)
    index = [(t // 37) % 4 - 1 for t in range(T)]
    check(ops.linear_adapters(x, w, ad, ops.AdapterRows(index, ad.ranks)), x, w, a, b, s, index)
    one = [1] * T
    check(ops.linear_adapters(x, w, ad, ops.AdapterRows(one, ad.ranks), torch.float32), x, w, a, b, s, one)


@pytest.mark.parametrize("T", [1, 3, 8, 12, 16, 40, 100, 150, 300])
def test_a_weight_that_the_call_before_makes(T):
    """A float32 weight filled by the kernel just before each product, new numbers every time and nothing between the calls: the
    products, which let the weights come before the activations in an engine, wait for it."""
    K, N, n = 512, 4096, 40
    g = torch.Generator("cuda").manual_seed(T)
    x = torch.randn((T, K), generator=g, device="cuda")
    ad = ops.Adapters(1, 16, N, K, torch.float32)
    rows = ops.AdapterRows([-1] * T, ad.ranks)
    w = torch.empty((N, K), device="cuda")
    calls = [lambda: ops.linear_adapters(x, w, ad, rows), lambda: ops.gemm_f32(x, w), lambda: ops.linear(x, w)]
    want = []
    for i in range(n):
        ops.fill_random(w, 1000 * T + i, 1.0)
        torch.cuda.synchronize()
        want.append(ops.gemm_f32(x, w))
        torch.cuda.synchronize()
    for call in calls:
        got = []
        for i in range(n):
            ops.fill_random(w, 1000 * T + i, 1.0)
            got.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("T", [1, 20, 70, 128, 200, 600])
def test_a_bfloat16_weight_that_the_call_before_makes(T):
    """The same with adapters, in each form of the bfloat16 product."""
    K, N, n = 1024, 4096, 40
    x, _, _, _, ad, _ = make(T, K, N, [16, 40], torch.bfloat16, T)
    rows = ops.AdapterRows([t % 3 - 1 for t in range(T)], ad.ranks)
    w = torch.empty((N, K), dtype=torch.bfloat16, device="cuda")
    want, got = [], []
    for i in range(n):
        ops.fill_random(w, 1000 * T + i, 1.0)
        torch.cuda.synchronize()
        want.append(ops.linear_adapters(x, w, ad, rows))
        torch.cuda.synchronize()
    for i in range(n):
        ops.fill_random(w, 1000 * T + i, 1.0)
        got.append(ops.linear_adapters(x, w, ad, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
