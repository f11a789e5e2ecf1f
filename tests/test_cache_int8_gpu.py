"""The cache of eight-bit rows and common prefixes, kernel by kernel, against 64 bits (GPU).

Tolerances.  A result is rounded to bfloat16 once: 2^-8 of it.  With A = sum_j p_j |v_j| per channel, a relative error e of the weights moves a result by at
most 2 e A (numerator and denominator).  A weight's own rounding is 2^-11 (half precision) or 2^-8 (bfloat16).  An error of a score moves its weight by as
much: the scores are sums of d products in float32 on tensor cores (2^-22 a step of S = scale sum_c |q_c k_jc|).  That bound adds every rounding up with one
sign; a second one, for the norm of the whole result, takes the two roundings to bfloat16 (weights, results) as independent: a rounding is off by 2^-8 / sqrt(12) on the average of its
range at most."""
import math
import subprocess
import sys

import pytest
import torch
from conftest import ROOT

from inferllm_b200.binding import KernelError

pytestmark = pytest.mark.gpu
B16, B8H, B8B = 2.0 ** -8, 2.0 ** -11, 2.0 ** -22


@pytest.fixture(scope="module")
def ops():
    from inferllm_b200.kernels import ops
    return ops


def take_error(ops):
    """The tensor-core kernels' error word, which goes back to 0."""
    torch.cuda.synchronize()
    word = ops.tc_error_word()
    value = int(word.item())
    word.zero_()
    return value


class Pages:
    """Sequences of given lengths on shuffled pages, some positions in common; what no sequence holds is unreadable (NaN scales)."""

    def __init__(self, seed, lens, nkv, d, page=64, common=None, int8=True, loud=3.0):
        g = torch.Generator().manual_seed(seed)
        common = common or [(0, None)] * len(lens)
        need = {}
        for i, (n, (c, a)) in enumerate(zip(lens, common)):
            assert c % page == 0 and c <= n
            for lp in range(-(-n // page)):
                need[(a, lp) if lp < c // page else (i, lp, "own")] = None
        self.pages = len(need) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        for key in need:
            need[key] = order.pop()
        width = max(-(-n // page) for n in lens) + 1
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        held = torch.zeros((self.pages, page), dtype=torch.bool)
        for i, (n, (c, a)) in enumerate(zip(lens, common)):
            for lp in range(-(-n // page)):
                p = need[(a, lp) if lp < c // page else (i, lp, "own")]
                self.table[i, lp] = p
                held[p, :max(0, min(page, n - lp * page))] = True
        shape = (self.pages, nkv, page, d)
        k = torch.randn(shape, generator=g)
        k[..., : max(1, d // 40)] *= loud
        v = torch.randn(shape, generator=g)
        self.lens, self.nkv, self.d, self.page, self.int8 = lens, nkv, d, page, int8
        hidden = ~held[:, None, :, None]
        if int8:
            def quantise(x):
                s = x.abs().amax(-1) / 127
                return (torch.round(x / s[..., None]) + 128).to(torch.uint8), s
            (self.ku, self.ks), (self.vu, self.vs) = quantise(k), quantise(v)
            for s in (self.ks, self.vs):
                s.masked_fill_(hidden[..., 0].expand_as(s), float("nan"))
        else:
            self.k, self.v = (x.bfloat16().masked_fill(hidden, float("nan")) for x in (k, v))

    def rows(self, seq):
        """Keys and values of a sequence in 64 bits, [n, nkv, d]."""
        n = self.lens[seq]
        at = self.table[seq, :-(-n // self.page)].long()

        def one(u, s=None):
            x = u[at].double()
            if s is not None:
                x = (x - 128) * s[at].double()[..., None]
            return x.transpose(1, 2).reshape(-1, self.nkv, self.d)[:n]
        return (one(self.ku, self.ks), one(self.vu, self.vs)) if self.int8 else (one(self.k), one(self.v))

    def cache(self, ops):
        if self.int8:
            return ops.CacheInt8(self.ku.cuda(), self.vu.cuda(), self.ks.cuda(), self.vs.cuda())
        return self.k.cuda(), self.v.cuda()


def first_visible(p, span):
    if span < 0:
        return p - p % -span
    return max(0, p - span + 1) if span > 0 else 0


def expected(pages, q, places, nh, span, scale, weight_error):
    """(results, tolerances) in 64 bits of queries q [T, nh * d] at places [(sequence, position)]."""
    out, tol = [], []
    G = nh // pages.nkv
    for t, (seq, p) in enumerate(places):
        k, v = pages.rows(seq)
        lo = first_visible(p, span)
        k, v = k[lo:p + 1], v[lo:p + 1]
        for h in range(nh):
            qh = q[t, h * pages.d:(h + 1) * pages.d].double()
            kh, vh = k[:, h // G], v[:, h // G]
            w = torch.softmax(kh @ qh * scale, 0)
            o = w @ vh
            absolute = scale * (kh.abs() @ qh.abs()).max()
            e = weight_error + absolute * (pages.d + 8) * B8B + (len(w) / 16 + 8) * B8B
            out.append(o)
            tol.append(B16 * o.abs() + 2 * e * (w @ vh.abs()) + 1e-42)
    return torch.stack(out).reshape(len(places), -1), torch.stack(tol).reshape(len(places), -1)


def near(got, want, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    worst = (off / tol).max()
    assert worst <= 1, f"{worst:.3g} times the tolerance"


def near_norm(got, want):
    """Two independent roundings to bfloat16 of relative size 2^-8 / sqrt(12) at most (twice that)."""
    rel = (got.double().cpu() - want).norm() / want.norm()
    assert rel <= 2 * math.sqrt(2) * B16 / math.sqrt(12), rel


def queries(seed, T, width, dtype=torch.bfloat16):
    return (torch.randn((T, width), generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype)


# ---------------------------------------------------------------- writing and reading

WRITES = [  # heads, kv heads, head size, rotated, page, tokens per sequence, dtype
    (32, 8, 128, 128, 64, [1], torch.bfloat16),
    (32, 8, 128, 128, 64, [5, 1, 130], torch.bfloat16),
    (4, 2, 64, 64, 64, [3, 64, 65], torch.bfloat16),
    (4, 2, 64, 32, 128, [7], torch.bfloat16),
    (6, 2, 24, 24, 7, [9, 20], torch.bfloat16),
    (3, 1, 80, 10, 16, [17], torch.bfloat16),
    (2, 2, 256, 64, 5, [11], torch.bfloat16),
    (5, 5, 8, 0, 3, [4, 4], torch.bfloat16),
    (4, 4, 16, 16, 16, [33], torch.float32),
    (6, 2, 24, 6, 7, [9, 20], torch.float32),
    (14, 2, 64, 64, 64, [200], torch.float32),
    (32, 32, 128, 128, 64, [700], torch.bfloat16),
]


def write_case(ops, seed, nh, nkv, d, rot, page, new, dtype, past=3):
    g = torch.Generator().manual_seed(seed)
    lens = [past + n for n in new]
    T = sum(new)
    x = torch.randn((T, nh + 2 * nkv, d), generator=g) * torch.exp(torch.randn((T, nh + 2 * nkv, 1), generator=g))
    if T > 2:
        x[1, nh:] = 0.0                         # rows of zeros
        x[2, nh:] *= 2.0 ** -110                # below what float32 scales can say
    qkv = x.reshape(T, -1).to(dtype)
    n_pos = max(lens)
    angle = torch.arange(n_pos, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, max(rot, 1), 2, dtype=torch.float64) / max(rot, 1))
    table = torch.stack([angle.cos(), angle.sin()], -1).float()
    pages = sum(-(-n // page) for n in lens) + 2
    order = torch.randperm(pages, generator=g).tolist()
    bt = torch.full((len(new), -(-max(lens) // page)), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for lp in range(-(-n // page)):
            bt[i, lp] = order.pop()
    seq = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], dtype=torch.int32)
    pos = torch.tensor([past + j for n in new for j in range(n)], dtype=torch.int32)
    cache = ops.CacheInt8.empty(pages, nkv, page, d)
    for t in (cache.k, cache.v):
        t.fill_(7)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(-1.0)
    return qkv, table if rot else None, bt, seq, pos, cache, torch.zeros(1, dtype=torch.int32, device="cuda")


def turned(qkv, table, pos, nh, nkv, d, rot):
    x = qkv.double().reshape(len(pos), nh + 2 * nkv, d).clone()
    if rot:
        at = table[pos.long()].double()[:, None]
        a, b = x[:, :nh + nkv, :rot // 2].clone(), x[:, :nh + nkv, rot // 2:rot].clone()
        x[:, :nh + nkv, :rot // 2] = a * at[..., 0] - b * at[..., 1]
        x[:, :nh + nkv, rot // 2:rot] = a * at[..., 1] + b * at[..., 0]
    return x


@pytest.mark.parametrize("nh, nkv, d, rot, page, new, dtype", WRITES)
@pytest.mark.parametrize("slices", [0, 3])
def test_rows_are_written_and_read_back(ops, nh, nkv, d, rot, page, new, dtype, slices):
    if slices and dtype != torch.bfloat16:
        pytest.skip("unreduced slices are the bfloat16 products'")
    qkv, table, bt, seq, pos, cache, err = write_case(ops, 5, nh, nkv, d, rot, page, new, dtype)
    given = qkv.cuda()
    if slices:
        ws = torch.randn((slices,) + tuple(qkv.shape), generator=torch.Generator().manual_seed(3)).cuda()
        ws[0] = given.float() - ws[1:].sum(0)
        given, qkv = ops.SplitKPartials(ws), ((ws[0] + ws[1]) + ws[2]).cpu()      # as the kernel adds
    dev = [t.cuda() for t in (pos, seq, bt)]
    q = ops.kv_write_int8(given, table.cuda() if rot else None, rot, *dev, cache, nh, err)
    assert int(err.item()) == 0
    x = turned(qkv, table, pos, nh, nkv, d, rot)
    # float32 sums of two products: three roundings of 2^-24 of their parts, which are below sqrt(2) max |x|
    fuzz = qkv.double().abs().reshape(len(pos), -1, d).amax(-1) * 3 * 2.0 ** -23
    got = q.double().cpu().reshape(len(pos), nh, d)
    unit = torch.finfo(dtype).eps / 2
    assert ((got - x[:, :nh]).abs() <= unit * x[:, :nh].abs() + fuzz[:, :nh, None] * 1.01).all()
    page_at = bt[seq.long(), (pos // page).long()].long()
    for u, s, rows, f in ((cache.k, cache.k_scale, x[:, nh:nh + nkv], fuzz[:, nh:nh + nkv]), (cache.v, cache.v_scale, x[:, nh + nkv:], fuzz[:, nh + nkv:])):
        u, s = u.cpu(), s.cpu()
        gu, gs = u[page_at, :, (pos % page).long()].double(), s[page_at, :, (pos % page).long()].double()
        top = rows.abs().amax(-1)
        tiny = top < 2.0 ** -99
        assert (gs[tiny] == 0).all() and (gu[tiny] == 128).all()
        assert ((gs - top / 127).abs() <= top * 2.0 ** -23 / 127 + f / 127)[~tiny].all()
        stands = (gu - 128) * gs[..., None]
        # half a step, and what moves a value across its border
        assert ((stands - rows).abs() <= (gs[..., None] / 2) * (1 + 2.0 ** -14) + f[..., None] * 2)[~tiny].all()
        assert (gu[~tiny].sub(128).abs().amax(-1) == 127).all()
        mark = torch.zeros(s.shape, dtype=torch.bool)
        mark[page_at, :, (pos % page).long()] = True
        assert (s[~mark] == -1).all() and (u[~mark] == 7).all()            # nothing else was touched
    for t in (torch.bfloat16, torch.float32):
        k, v = ops.kv_read_int8(cache, *dev, dtype=t)
        for back, u, s in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
            p = (pos % page).long().cuda()
            want = (u[page_at.cuda(), :, p].float() - 128) * s[page_at.cuda(), :, p][..., None]
            assert torch.equal(back, want.to(t))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_that_is_not_finite_reads_back_as_nan(ops, bad, dtype):
    nh, nkv, d, page = 4, 2, 64, 64
    qkv, table, bt, seq, pos, cache, err = write_case(ops, 5, nh, nkv, d, d, page, [6], dtype)
    x = qkv.reshape(6, nh + 2 * nkv, d)
    x[4, nh + 1, 3] = bad                  # a key of kv head 1
    x[5, nh + nkv, 63] = bad               # a value of kv head 0
    dev = [t.cuda() for t in (pos, seq, bt)]
    ops.kv_write_int8(qkv.cuda(), table.cuda(), d, *dev, cache, nh, err)
    k, v = ops.kv_read_int8(cache, *dev, dtype=torch.float32)
    want_k, want_v = torch.zeros(6, nkv, dtype=torch.bool), torch.zeros(6, nkv, dtype=torch.bool)
    want_k[4, 1] = True
    want_v[5, 0] = True
    assert torch.equal(torch.isnan(k).cpu(), want_k[..., None].expand(6, nkv, d)) and torch.equal(torch.isnan(v).cpu(), want_v[..., None].expand(6, nkv, d))


def test_positions_without_a_page_or_beyond_the_table(ops):
    nh, nkv, d, page = 4, 2, 64, 64
    qkv, table, bt, seq, pos, cache, err = write_case(ops, 5, nh, nkv, d, d, page, [3, 2], torch.bfloat16)
    bt[1, 0] = -1
    before = cache.k_scale.clone()
    ops.kv_write_int8(qkv.cuda(), table.cuda(), d, pos.cuda(), seq.cuda(), bt.cuda(), cache, nh, err)
    assert int(err.item()) == 2
    assert int((cache.k_scale != before).sum()) == 3 * nkv
    err.zero_()
    for wrong in (bt.clone().fill_(cache.pages), bt.clone().fill_(2 ** 31 - 1)):
        ops.kv_write_int8(qkv.cuda(), table.cuda(), d, pos.cuda(), seq.cuda(), wrong.cuda(), cache, nh, err)
        assert int(err.item()) == 2
    err.zero_()
    bt[1, 0] = 0 if int(bt[0, 0]) else 1
    far = pos.clone()
    far[4] = len(table)
    ops.kv_write_int8(qkv.cuda(), table.cuda(), d, far.cuda(), seq.cuda(), bt.cuda(), cache, nh, err)
    assert int(err.item()) == 3
    far[4] = 10 ** 6                          # beyond the block table's width too
    k, _ = ops.kv_read_int8(cache, far.cuda(), seq.cuda(), bt.cuda())
    assert torch.isnan(k[4]).all() and not torch.isnan(k[:4]).any()
    far[4] = -1
    k, _ = ops.kv_read_int8(cache, far.cuda(), seq.cuda(), bt.cuda())
    assert torch.isnan(k[4]).all()


# ---------------------------------------------------------------- single tokens

SINGLE = [  # heads, kv heads, head size, page, lengths, window
    (32, 8, 128, 64, [1], 0),
    (32, 8, 128, 64, [777], 0),
    (4, 2, 64, 64, [64, 65, 1, 63, 300], 0),
    (14, 2, 64, 128, [500, 129, 128], 0),
    (16, 1, 128, 64, [200, 17], 0),
    (8, 8, 128, 192, [193, 400], 0),
    (3, 3, 64, 64, [90, 15, 16, 33], 0),
    (8, 2, 128, 64, [500, 70, 3], 100),
    (8, 2, 64, 64, [500, 70, 3], 1),
    (8, 2, 64, 64, [500, 129, 128, 127], -128),
    (8, 2, 128, 64, [500, 77], 10000),
]


@pytest.mark.parametrize("nh, nkv, d, page, lens, window", SINGLE)
@pytest.mark.parametrize("splits", [None, 1, 3, 32])
def test_single_tokens(ops, nh, nkv, d, page, lens, window, splits):
    pages = Pages(11, lens, nkv, d, page)
    T, scale = len(lens), d ** -0.5
    q = queries(7, T, (nh + 2 * nkv) * d)                 # rows of a packed projection: the queries come first
    places = [(i, n - 1) for i, n in enumerate(lens)]
    want, tol = expected(pages, q, places, nh, window, scale, B8H)
    pos, seq = torch.tensor([p for _, p in places], dtype=torch.int32).cuda(), torch.arange(T, dtype=torch.int32).cuda()
    got = ops.attention_decode_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, nh, window, scale, max(lens), splits=splits)
    near(got, want, tol)
    assert take_error(ops) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh, nkv, d, page, lens, window", [
    (6, 2, 24, 7, [1, 8, 40], 0), (4, 4, 16, 16, [33, 16], 0), (34, 2, 64, 64, [70, 5], 0), (2, 1, 256, 5, [21], 0), (4, 1, 80, 64, [130], 20), (4, 2, 8, 3, [50], -16),
    (4, 2, 128, 32, [100, 31], 0)])
def test_single_tokens_of_other_sizes(ops, nh, nkv, d, page, lens, window, dtype):
    pages = Pages(13, lens, nkv, d, page)
    T, scale = len(lens), d ** -0.5
    q = queries(7, T, nh * d, dtype)
    places = [(i, n - 1) for i, n in enumerate(lens)]
    # float32 throughout: exp2f within two units, sums of up to 256 products and a few hundred weights
    want, tol = expected(pages, q, places, nh, window, scale, 8 * 2.0 ** -23)
    if dtype == torch.float32:
        tol = tol - B16 * want.abs() + 2.0 ** -23 * want.abs()
    pos, seq = torch.tensor([p for _, p in places], dtype=torch.int32).cuda(), torch.arange(T, dtype=torch.int32).cuda()
    got = ops.attention_decode_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, nh, window, scale, max(lens))
    assert got.dtype == dtype
    near(got, want, tol)
    assert take_error(ops) == 0


@pytest.mark.parametrize("power", [-100, -30, 20, 60, 100])
def test_scales_of_any_size(ops, power):
    """Values times a power of two: the results are multiplied by it.  Scores too, through the keys, as far as they stay scores."""
    pages = Pages(17, [300, 64], 2, 128)
    q, scale = queries(3, 2, 8 * 128), 128 ** -0.5
    pos, seq = torch.tensor([299, 63], dtype=torch.int32).cuda(), torch.arange(2, dtype=torch.int32).cuda()
    pages.vs *= 2.0 ** power
    pages.ks *= 2.0 ** -power
    want, tol = expected(pages, q, [(0, 299), (1, 63)], 8, 0, scale * 2.0 ** power, B8H)
    got = ops.attention_decode_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, 8, 0, scale * 2.0 ** power, 300)
    near(got, want, tol)


@pytest.mark.parametrize("power", [-100, 100])
def test_scales_of_any_size_on_wide_tiles(ops, power):
    """The same for prompts and for a common prefix of many rows, whose weights carry the values' scales in bfloat16's range."""
    nh, nkv, d, n = 8, 2, 128, 20
    lens = [150 + i for i in range(n)]
    pages = Pages(17, lens, nkv, d, common=[(128, 0)] * n)
    pages.vs *= 2.0 ** power
    pages.ks *= 2.0 ** -power
    scale = d ** -0.5 * 2.0 ** power
    pos, seq = torch.tensor(lens, dtype=torch.int32).cuda() - 1, torch.arange(n, dtype=torch.int32).cuda()
    q = queries(3, n, nh * d)
    want, tol = expected(pages, q, [(i, m - 1) for i, m in enumerate(lens)], nh, 0, scale, B16)
    plan = ops.SharedPrefixes([(128, list(range(n)))], lens, nh // nkv)
    assert plan.wide
    near(ops.attention_decode_shared(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, plan, nh, scale, max(lens)), want, tol)
    cu = torch.arange(0, n + 1, dtype=torch.int32).cuda()
    near(ops.attention_prompts_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), cu, pos + 1, 1, nh, 0, scale), want, tol)
    assert take_error(ops) == 0


def test_launches_that_wait_for_the_whole_of_the_one_before(ops):
    """Without programmatic launches the kernels of a call follow one another: the same bits."""
    nh, nkv, d, n = 8, 2, 64, 40
    lens = [300 + 3 * i for i in range(n)]
    pages = Pages(23, lens, nkv, d, common=[(256, 0)] * n)
    pos, seq = torch.tensor(lens, dtype=torch.int32).cuda() - 1, torch.arange(n, dtype=torch.int32).cuda()
    q, cache, table = queries(5, n, nh * d).cuda(), pages.cache(ops), pages.table.cuda()
    for groups in ([(256, list(range(n)))], [(256, list(range(i, i + 4))) for i in range(0, n, 4)]):
        plan = ops.SharedPrefixes(groups, lens, nh // nkv)
        got = []
        try:
            for on in (True, False):
                ops.set_pdl(on)
                got.append([ops.attention_decode_shared(q, cache, table, pos, seq, plan, nh, 0.1, max(lens)) for _ in range(3)])
                torch.cuda.synchronize()
        finally:
            ops.set_pdl(True)
        assert all(torch.equal(got[0][0], g) for row in got for g in row)
    assert take_error(ops) == 0


def test_queries_of_any_size(ops):
    for power in (-120, -60, 60, 100):
        pages = Pages(17, [300, 64], 2, 64)
        q = queries(3, 2, 8 * 64)
        scale = 64 ** -0.5 * 2.0 ** -power
        big = (q.double() * 2.0 ** power).bfloat16()
        want, tol = expected(pages, q, [(0, 299), (1, 63)], 8, 0, 64 ** -0.5, B8H)
        pos, seq = torch.tensor([299, 63], dtype=torch.int32).cuda(), torch.arange(2, dtype=torch.int32).cuda()
        got = ops.attention_decode_int8(big.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, 8, 0, scale, 300)
        near(got, want, tol)


def test_values_of_unequal_sizes(ops):
    """One key of tiny weight with huge values next to many of ordinary ones, and the other way round."""
    pages = Pages(19, [200], 1, 64)
    at = pages.table[0].long()
    pages.vs[at[0], 0, 5] *= 2.0 ** 20
    pages.vs[at[1], 0, 7] *= 2.0 ** -40
    pages.vs[at[2], 0, 0] = 0.0
    pages.ks[at[2], 0, 1] = 0.0
    q = queries(23, 1, 4 * 64)
    want, tol = expected(pages, q, [(0, 199)], 4, 0, 0.125, B8H)
    got = ops.attention_decode_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), torch.tensor([199], dtype=torch.int32).cuda(),
                                    torch.zeros(1, dtype=torch.int32).cuda(), 4, 0, 0.125, 200)
    near(got, want, tol)


@pytest.mark.parametrize("d, dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (24, torch.bfloat16), (64, torch.float32)])
def test_rows_that_are_not_numbers_reach_who_sees_them(ops, d, dtype):
    nh, nkv, lens = 4, 2, [150, 150, 40]
    pages = Pages(29, lens, nkv, d)
    q = queries(31, 3, nh * d, dtype)
    want, _ = expected(pages, q, [(i, n - 1) for i, n in enumerate(lens)], nh, 0, d ** -0.5, 0.0)
    clean = want.reshape(3, nh, d)
    pages.ks[pages.table[0, 1].long(), 0, 3] = float("nan")        # a key of sequence 0, kv head 0
    pages.vs[pages.table[1, 2].long(), 1, 21] = float("nan")       # a value of sequence 1, kv head 1: position 149, its last one
    pos, seq = torch.tensor([n - 1 for n in lens], dtype=torch.int32).cuda(), torch.arange(3, dtype=torch.int32).cuda()
    got = ops.attention_decode_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, nh, 0, d ** -0.5, 150).reshape(3, nh, d).float().cpu()
    nan = torch.zeros((3, nh), dtype=torch.bool)
    nan[0, :2] = True
    nan[1, 2:] = True
    assert torch.equal(torch.isnan(got).all(-1), nan) and torch.equal(torch.isnan(got).any(-1), nan)
    assert (got[~nan].double() - clean[~nan]).norm() <= 0.01 * clean[~nan].norm()


@pytest.mark.parametrize("kind", ["tensor cores", "plain"])
def test_a_token_without_a_position_gets_zeros(ops, kind):
    d = 64 if kind == "tensor cores" else 32
    pages = Pages(37, [100, 100], 2, d)
    q = queries(41, 2, 4 * d).cuda()
    pos = torch.tensor([-1, 99], dtype=torch.int32).cuda()
    for splits in (1, 4):
        got = ops.attention_decode_int8(q, pages.cache(ops), pages.table.cuda(), pos, torch.arange(2, dtype=torch.int32).cuda(), 4, 0, 0.1, 100, splits=splits)
        assert (got[0] == 0).all() and torch.isfinite(got).all() and (got[1] != 0).any()


@pytest.mark.parametrize("d", [64, 32])
def test_a_page_that_is_not_held_is_reported(ops, d):
    """Nothing outside the pages is read: the kernels look before they load."""
    pages = Pages(43, [200, 100], 2, d)
    q, seq = queries(47, 2, 4 * d).cuda(), torch.arange(2, dtype=torch.int32).cuda()
    cache, table = pages.cache(ops), pages.table
    pos = torch.tensor([199, 99], dtype=torch.int32).cuda()
    assert take_error(ops) == 0
    for bad in (-1, pages.pages, -2 ** 31, 2 ** 31 - 1):
        wrong = table.clone()
        wrong[0, 1] = bad
        ops.attention_decode_int8(q, cache, wrong.cuda(), pos, seq, 4, 0, 0.1, 200)
        assert take_error(ops) == 8
    far = torch.tensor([199, 64 * table.shape[1]], dtype=torch.int32).cuda()       # beyond the block table
    ops.attention_decode_int8(q, cache, table.cuda(), far, seq, 4, 0, 0.1, 64 * table.shape[1] + 1)
    assert take_error(ops) == 8


# ---------------------------------------------------------------- prompts

PROMPTS = [  # heads, kv heads, head size, page, new tokens, past, window
    (4, 2, 64, 64, [1], [0], 0),
    (4, 2, 64, 64, [200], [0], 0),
    (32, 8, 128, 64, [70], [0], 0),
    (8, 8, 128, 64, [300, 1, 129], [0, 5, 64], 0),
    (14, 2, 64, 128, [40, 130], [100, 63], 0),
    (16, 1, 128, 64, [33, 2], [1, 300], 0),
    (6, 2, 64, 64, [257, 256], [0, 0], 0),
    (4, 2, 128, 64, [300, 50], [0, 200], 70),
    (2, 2, 64, 64, [400], [100], 1),
    (4, 1, 128, 64, [300, 90], [37, 0], -100),
    (4, 2, 64, 64, [0, 65, 0], [7, 0, 0], 0),
]


@pytest.mark.parametrize("nh, nkv, d, page, new, past, window", PROMPTS)
@pytest.mark.parametrize("tile_rows", [128, 256])
def test_prompts(ops, nh, nkv, d, page, new, past, window, tile_rows):
    lens = [max(1, p + n) for p, n in zip(past, new)]
    pages = Pages(53, lens, nkv, d, page)
    T, scale = sum(new), d ** -0.5
    q = queries(59, T, (nh + 2 * nkv) * d)
    places = [(i, p + j) for i, (p, n) in enumerate(zip(past, new)) for j in range(n)]
    want, tol = expected(pages, q, places, nh, window, scale, B16)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32).cuda()
    got = ops.attention_prompts_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), cu, torch.tensor([p + n for p, n in zip(past, new)], dtype=torch.int32).cuda(),
                                     max(new), nh, window, scale, tile_rows=tile_rows)
    near(got, want, tol)
    near_norm(got, want)
    assert take_error(ops) == 0


def test_prompt_rows_before_the_first_position_are_zeros(ops):
    """A sequence said to be shorter than its new tokens: those before position 0 see nothing (of the first 40, 20 and 260 tokens a part of a tile, and more
    than a tile of two sequences' heads)."""
    nh, nkv, d, scale = 4, 2, 64, 0.125
    new, lens = [100, 30, 300], [60, 10, 40]
    pages = Pages(71, lens, nkv, d)
    T = sum(new)
    q = queries(73, T, nh * d)
    cu = torch.tensor([0, 100, 130, 430], dtype=torch.int32).cuda()
    for tile_rows in (128, 256):
        got = ops.attention_prompts_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), cu, torch.tensor(lens, dtype=torch.int32).cuda(), 300, nh, 0, scale, tile_rows=tile_rows)
        assert take_error(ops) == 0
        for i, (n, length) in enumerate(zip(new, lens)):
            first = sum(new[:i])
            assert (got[first:first + n - length] == 0).all()
            mine = slice(first + n - length, first + n)
            want, tol = expected(pages, q[mine], [(i, j) for j in range(length)], nh, 0, scale, B16)
            near(got[mine], want, tol)

def test_a_row_that_is_not_a_number_reaches_later_queries_only(ops):
    nh, nkv, d, n = 4, 2, 64, 150
    for which in ("k", "v"):
        pages = Pages(61, [n], nkv, d)
        q = queries(67, n, nh * d)
        want, _ = expected(pages, q, [(0, j) for j in range(n)], nh, 0, 0.125, 0.0)
        (pages.ks if which == "k" else pages.vs)[pages.table[0, 1].long(), 1, 6] = float("nan")        # position 70, kv head 1
        got = ops.attention_prompts_int8(q.cuda(), pages.cache(ops), pages.table.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(),
                                         torch.tensor([n], dtype=torch.int32).cuda(), n, nh, 0, 0.125).reshape(n, nh, d).float().cpu()
        nan = torch.zeros((n, nh), dtype=torch.bool)
        nan[70:, 2:] = True
        assert torch.equal(torch.isnan(got).all(-1), nan) and torch.equal(torch.isnan(got).any(-1), nan)
        ok = want.reshape(n, nh, d)[~nan]
        assert (got[~nan].double() - ok).norm() <= 0.01 * ok.norm()


def test_prompts_on_a_page_that_is_not_held(ops):
    pages = Pages(43, [200], 2, 64)
    q = queries(47, 30, 4 * 64).cuda()
    args = torch.tensor([0, 30], dtype=torch.int32).cuda(), torch.tensor([200], dtype=torch.int32).cuda(), 30, 4, 0, 0.1
    for bad in (-1, pages.pages, 2 ** 31 - 1):
        wrong = pages.table.clone()
        wrong[0, 1] = bad
        ops.attention_prompts_int8(q, pages.cache(ops), wrong.cuda(), *args)
        assert take_error(ops) == 8
    ops.attention_prompts_int8(q, pages.cache(ops), pages.table[:, :2].contiguous().cuda(), *args)
    assert take_error(ops) == 8


# ---------------------------------------------------------------- positions in common

SHARED = [  # heads, kv heads, head size, page, per sequence (length, prefix, group)
    (32, 8, 128, 64, [(200, 128, 0), (129, 128, 0)]),
    (4, 4, 64, 64, [(70, 64, 0)] * 9 + [(100, 0, None)]),
    (8, 2, 128, 64, [(300 + i, 256, 0) for i in range(40)]),
    (14, 2, 64, 128, [(260, 256, 0), (400, 128, 1), (129, 128, 1), (50, 0, None), (300, 256, 0)]),
    (16, 1, 128, 64, [(150 + 10 * i, 64 * (1 + i % 2), i % 2) for i in range(35)]),
    (6, 2, 64, 64, [(128, 128, 0), (128, 128, 0), (128, 128, 0)]),
    (8, 8, 128, 64, [(500 + i, 448, 0) for i in range(33)]),
    (8, 2, 64, 64, [(3, 0, None), (90, 0, None)]),
]


@pytest.mark.parametrize("nh, nkv, d, page, seqs", SHARED)
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("own, pre", [(None, None), (1, 1), (3, 5), (32, 32)])
def test_positions_in_common(ops, nh, nkv, d, page, seqs, int8, own, pre):
    lens = [n for n, _, _ in seqs]
    pages = Pages(71, lens, nkv, d, page, common=[(c, "g%s" % a) for _, c, a in seqs], int8=int8)
    T, scale = len(seqs), d ** -0.5
    q = queries(73, T, (nh + 2 * nkv) * d)
    groups = {}
    for t, (_, c, a) in enumerate(seqs):
        if a is not None:
            groups.setdefault((c, a), []).append(t)
    plan = ops.SharedPrefixes([(c, m[::-1]) for (c, _), m in groups.items()], lens, nh // nkv)
    places = [(i, n - 1) for i, n in enumerate(lens)]
    want, tol = expected(pages, q, places, nh, 0, scale, B8H if int8 and not plan.wide else B16)
    pos, seq = torch.tensor([p for _, p in places], dtype=torch.int32).cuda(), torch.arange(T, dtype=torch.int32).cuda()
    got = ops.attention_decode_shared(q.cuda(), pages.cache(ops), pages.table.cuda(), pos, seq, plan, nh, scale, max(lens), own_splits=own, pre_splits=pre)
    near(got, want, tol)
    near_norm(got, want)
    assert take_error(ops) == 0


def test_a_prefix_that_ends_inside_a_page(ops):
    """The plan may leave more to the tokens than their pages have in common: what counts is what it says."""
    seqs = [(300, 192, 0)] * 20
    for int8 in (True, False):
        pages = Pages(79, [300] * 20, 2, 64, common=[(192, "g")] * 20, int8=int8)
        q = queries(83, 20, 8 * 64)
        want, tol = expected(pages, q, [(i, 299) for i in range(20)], 8, 0, 0.125, B16)
        for prefix, members in ((1, 20), (63, 20), (130, 3), (100, 20)):
            plan = ops.SharedPrefixes([(prefix, list(range(members)))], [300] * 20, 4)
            got = ops.attention_decode_shared(q.cuda(), pages.cache(ops), pages.table.cuda(), torch.full((20,), 299, dtype=torch.int32).cuda(),
                                              torch.arange(20, dtype=torch.int32).cuda(), plan, 8, 0.125, 300)
            near(got, want, tol)
    assert len(seqs) == 20 and take_error(ops) == 0


# ---------------------------------------------------------------- together, streams, graphs, refusals


def test_written_then_attended(ops):
    """A prompt and two single tokens behind it, as a layer does it: rotate and write, then attend, against 64 bits of the same rows."""
    nh, nkv, d, page = 8, 2, 128, 64
    new, steps = [70, 130], 2
    lens = [n + steps for n in new]
    g = torch.Generator().manual_seed(89)
    angle = torch.arange(max(lens), dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    table = torch.stack([angle.cos(), angle.sin()], -1).float()
    bt = torch.tensor([[3, 1, 7], [0, 5, 2]], dtype=torch.int32).cuda()
    cache, err = ops.CacheInt8.empty(8, nkv, page, d), torch.zeros(1, dtype=torch.int32, device="cuda")
    for s in (cache.k_scale, cache.v_scale):
        s.fill_(float("nan"))
    past = [0, 0]
    for step in range(steps + 1):
        n = new if step == 0 else [1, 1]
        seq = torch.tensor([i for i, c in enumerate(n) for _ in range(c)], dtype=torch.int32)
        pos = torch.tensor([past[i] + j for i, c in enumerate(n) for j in range(c)], dtype=torch.int32)
        qkv = torch.randn((len(pos), (nh + 2 * nkv) * d), generator=g).bfloat16()
        q = ops.kv_write_int8(qkv.cuda(), table.cuda(), d, pos.cuda(), seq.cuda(), bt, cache, nh, err)
        past = [p + c for p, c in zip(past, n)]
        if step == 0:
            cu = torch.tensor([0, n[0], sum(n)], dtype=torch.int32).cuda()
            got = ops.attention_prompts_int8(q, cache, bt, cu, torch.tensor(past, dtype=torch.int32).cuda(), max(n), nh, 0, d ** -0.5)
        else:
            got = ops.attention_decode_int8(q, cache, bt, pos.cuda(), seq.cuda(), nh, 0, d ** -0.5, max(lens))
        held = Pages.__new__(Pages)
        held.ku, held.vu, held.ks, held.vs = (t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))
        held.table, held.lens, held.nkv, held.d, held.page, held.int8 = bt.cpu(), past, nkv, d, page, True
        want, tol = expected(held, q.cpu(), list(zip(seq.tolist(), pos.tolist())), nh, 0, d ** -0.5, B16 if step == 0 else B8H)
        near(got, want, tol)
    assert int(err.item()) == 0 and take_error(ops) == 0


def test_on_another_stream_and_captured(ops):
    nh, nkv, d = 8, 2, 64
    seqs = [(300 + i, 256, 0) for i in range(12)]
    lens = [n for n, _, _ in seqs]
    pages = Pages(97, lens, nkv, d, common=[(256, "g")] * 12)
    cache, table = pages.cache(ops), pages.table.cuda()
    pos, seq = torch.tensor([n - 1 for n in lens], dtype=torch.int32).cuda(), torch.arange(12, dtype=torch.int32).cuda()
    plan = ops.SharedPrefixes([(256, list(range(12)))], lens, 4)
    cu, after = torch.arange(13, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q = queries(101, 12, nh * d).cuda()

    def calls(x):
        return (ops.attention_decode_int8(x, cache, table, pos, seq, nh, 0, 0.125, 400, splits=4), ops.attention_prompts_int8(x, cache, table, cu, after, 1, nh, 0, 0.125),
                ops.attention_decode_shared(x, cache, table, pos, seq, plan, nh, 0.125, 400, own_splits=2, pre_splits=3))
    want, other = calls(q), calls(q * 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = calls(q)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two graphs, replayed in turn and then side by side: neither has the other's scratch
    graphs = []
    for x in (q, q * 2):
        graph, static = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph):
            out = calls(static)
        graphs.append((graph, static, out))
    for _ in range(2):
        for graph, _, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_, _, out), w in zip(graphs, (want, other)):
        assert all(torch.equal(a, b) for a, b in zip(w, out))
    for _, _, out in graphs:
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    for (_, _, out), w in zip(graphs, (want, other)):
        assert all(torch.equal(a, b) for a, b in zip(w, out))
    assert take_error(ops) == 0


def test_two_calls_at_once(ops):
    """Calls on two streams, none of which waits for the other, have scratch of their own: each gives what it gives alone."""
    nh, nkv, d, n = 32, 8, 128, 40
    lens = [600 + 7 * i for i in range(n)]
    pages = Pages(91, lens, nkv, d, common=[(512, 0)] * n)
    cache, table = pages.cache(ops), pages.table.cuda()
    pos, seq = torch.tensor(lens, dtype=torch.int32).cuda() - 1, torch.arange(n, dtype=torch.int32).cuda()
    plan = ops.SharedPrefixes([(512, list(range(n)))], lens, nh // nkv)
    q = [queries(s, n, nh * d).cuda() for s in (93, 97)]
    cu, ln = torch.arange(0, n + 1, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    runs = [lambda x: ops.attention_decode_shared(x, cache, table, pos, seq, plan, nh, 0.09, max(lens)),
            lambda x: ops.attention_decode_int8(x, cache, table, pos, seq, nh, 0, 0.09, max(lens), splits=16),
            lambda x: ops.attention_decode_int8(x, cache, table, pos, seq, nh, 0, 0.09, max(lens), splits=4),
            lambda x: ops.attention_prompts_int8(x, cache, table, cu, ln, 1, nh, 0, 0.09)]
    for run in runs:
        alone = [run(x) for x in q]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in q]
        got = [[], []]
        for _ in range(4):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(run(q[i]))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(alone[i], g) for g in got[i])
    assert take_error(ops) == 0


def test_more_tokens_than_a_grid_has_rows(ops):
    """65,540 single tokens go in two launches."""
    lens = [1, 70, 129]
    pages = Pages(101, lens, 1, 64)
    few = queries(103, 3, 64)
    T = 65540
    seq = (torch.arange(T) % 3).int()
    args = pages.cache(ops), pages.table.cuda()
    last = torch.tensor(lens, dtype=torch.int32) - 1
    got = ops.attention_decode_int8(few[seq.long()].contiguous().cuda(), *args, last[seq.long()].cuda(), seq.cuda(), 1, 0, 0.125, 129, splits=2)
    want = ops.attention_decode_int8(few.cuda(), *args, last.cuda(), torch.arange(3, dtype=torch.int32).cuda(), 1, 0, 0.125, 129, splits=2)
    assert torch.equal(got, want[seq.long().cuda()])
    assert take_error(ops) == 0


def test_the_same_call_gives_the_same_bits(ops):
    pages = Pages(103, [700, 300], 2, 128)
    q = queries(107, 2, 8 * 128).cuda()
    pos, seq = torch.tensor([699, 299], dtype=torch.int32).cuda(), torch.arange(2, dtype=torch.int32).cuda()
    cache, table = pages.cache(ops), pages.table.cuda()
    first = ops.attention_decode_int8(q, cache, table, pos, seq, 8, 0, 0.1, 700)
    for _ in range(5):
        assert torch.equal(first, ops.attention_decode_int8(q, cache, table, pos, seq, 8, 0, 0.1, 700))


def test_no_tokens(ops):
    cache = ops.CacheInt8.empty(2, 2, 64, 64)
    none, table = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    empty = torch.zeros((0, 8 * 64), dtype=torch.bfloat16, device="cuda")
    assert ops.attention_decode_int8(empty[:, :256], cache, table, none, none, 4, 0, 0.1, 1).shape == (0, 256)
    assert ops.kv_read_int8(cache, none, none, table)[0].shape == (0, 2, 64)
    assert ops.kv_write_int8(empty, None, 0, none, none, table, cache, 4, torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 256)
    cu, lens = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    assert ops.attention_prompts_int8(empty[:, :256], cache, table, cu, lens, 0, 4, 0, 0.1).shape == (0, 256)


def test_refusals(ops):
    cache = ops.CacheInt8.empty(3, 2, 64, 64)
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    pos, seq = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")
    q = torch.zeros((2, 4 * 64), dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def decode(**w):
        a = dict(q=q, cache=cache, block_table=table, token_pos=pos, token_seq=seq, n_heads=4, window=0, scale=0.1, max_len=10)
        return ops.attention_decode_int8(**{**a, **w})
    wrong = [dict(q=q.cpu()), dict(q=q.half()), dict(q=q[:, :200]), dict(q=q[0]), dict(n_heads=3), dict(n_heads=0), dict(token_pos=pos[:1]), dict(token_pos=pos.long()),
             dict(token_seq=seq.cpu()), dict(block_table=table[0]), dict(block_table=table.cpu()), dict(block_table=table[:, :0]), dict(max_len=0),
             dict(cache=(cache.k, cache.v)), dict(splits=33), dict(splits=0),
             dict(q=torch.zeros((2, 4 * 64 + 4), dtype=torch.bfloat16, device="cuda")), dict(q=torch.zeros(2 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 256)),
             dict(q=torch.zeros((256, 2), dtype=torch.bfloat16, device="cuda").t())]
    for w in wrong:
        with pytest.raises(KernelError):
            decode(**w)
    for make in (lambda: ops.CacheInt8(cache.k, cache.v[:2], cache.k_scale, cache.v_scale), lambda: ops.CacheInt8(cache.k.char(), cache.v, cache.k_scale, cache.v_scale),
                 lambda: ops.CacheInt8(cache.k, cache.v, cache.k_scale[:, :1].contiguous(), cache.v_scale), lambda: ops.CacheInt8(cache.k, cache.v, cache.k_scale.half(), cache.v_scale),
                 lambda: ops.CacheInt8(cache.k.cpu(), cache.v, cache.k_scale, cache.v_scale), lambda: ops.CacheInt8.empty(3, 2, 64, 12), lambda: ops.CacheInt8.empty(3, 2, 64, 264),
                 lambda: ops.CacheInt8.empty(0, 2, 64, 64), lambda: ops.CacheInt8.empty(3, 2, 64, 64, device="cpu")):
        with pytest.raises(KernelError):
            make()
    qkv = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device="cuda")
    cs = torch.zeros((9, 32, 2), device="cuda")
    for args in ((qkv[:, :448].contiguous(), cs, 64), (qkv, cs, 32), (qkv, cs, 66), (qkv, cs, 63), (qkv, None, 64), (qkv, cs.half(), 64), (qkv.half(), cs, 64), (qkv.cpu(), cs, 64)):
        with pytest.raises(KernelError):
            ops.kv_write_int8(*args, pos, seq, table, cache, 4, err)
    with pytest.raises(KernelError):
        ops.kv_write_int8(qkv, cs, 64, pos, seq, table, (cache.k, cache.v), 4, err)
    cu, lens = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    small = ops.CacheInt8.empty(3, 2, 64, 32)
    for args in ((q, small, table, cu, lens, 1, 4), (q.float(), cache, table, cu, lens, 1, 4), (q, cache, table, cu[:2], lens, 1, 4), (q, cache, table, cu, lens, 3, 4),
                 (q, cache, table, cu, lens, -1, 4), (q, ops.CacheInt8.empty(3, 2, 32, 64), table, cu, lens, 1, 4)):
        with pytest.raises(KernelError):
            ops.attention_prompts_int8(*args, 0, 0.1)
    plan = ops.SharedPrefixes([(64, [0, 1])], [65, 70], 2)
    for w in (dict(plan=ops.SharedPrefixes([(64, [0, 1])], [65, 70], 1)), dict(plan=ops.SharedPrefixes([], [65], 2)), dict(q=q.float()), dict(max_len=69), dict(cache=small),
              dict(cache=(cache.k, cache.v)), dict(cache=(cache.k.bfloat16(), cache.v.bfloat16()[:2])), dict(own_splits=33), dict(pre_splits=0), dict(pre_splits=33)):
        a = dict(q=q, cache=cache, block_table=table, token_pos=pos, token_seq=seq, plan=plan, n_heads=4, scale=0.1, max_len=70)
        with pytest.raises(KernelError):
            ops.attention_decode_shared(**{**a, **w})
    torch.cuda.synchronize()


def test_positions_beyond_32_bits_of_elements(ops):
    """Pages whose elements are numbered beyond 2^31: rows are found by 64-bit offsets."""
    pages, nkv, d = 2 ** 31 // (64 * 8 * 128) + 40, 8, 128
    cache = ops.CacheInt8.empty(pages, nkv, 64, d)
    last = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32).cuda()
    pos, seq = torch.arange(100, dtype=torch.int32).cuda(), torch.zeros(100, dtype=torch.int32).cuda()
    qkv, err = queries(109, 100, 48 * d).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = ops.kv_write_int8(qkv, None, 0, pos, seq, last, cache, 32, err)
    small = ops.CacheInt8.empty(2, nkv, 64, d)
    first = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    ops.kv_write_int8(qkv, None, 0, pos, seq, first, small, 32, err)
    for a, b in zip(ops.kv_read_int8(cache, pos, seq, last), ops.kv_read_int8(small, pos, seq, first)):
        assert torch.equal(a, b)
    one = (pos[99:], seq[99:])
    assert torch.equal(ops.attention_decode_int8(q[99:], cache, last, *one, 32, 0, 0.1, 100), ops.attention_decode_int8(q[99:], small, first, *one, 32, 0, 0.1, 100))
    cu, lens = torch.tensor([0, 100], dtype=torch.int32).cuda(), torch.tensor([100], dtype=torch.int32).cuda()
    assert torch.equal(ops.attention_prompts_int8(q, cache, last, cu, lens, 100, 32, 0, 0.1), ops.attention_prompts_int8(q, small, first, cu, lens, 100, 32, 0, 0.1))
    f = q[99:].float()
    assert torch.equal(ops.attention_decode_int8(f, cache, last, *one, 32, 0, 0.1, 100), ops.attention_decode_int8(f, small, first, *one, 32, 0, 0.1, 100))
    assert int(err.item()) == 0 and take_error(ops) == 0


def test_what_a_call_reads_stays_as_it_was_made(ops):
    """Addresses are taken once: another tensor in place of one that they belong to is refused, and one that is pointed elsewhere keeps its memory for the calls."""
    k, v = (torch.full((3, 2, 64, 64), 128 + i, dtype=torch.uint8, device="cuda") for i in (3, 5))
    ks, vs = (torch.ones((3, 2, 64), device="cuda") for _ in range(2))
    cache = ops.CacheInt8(k, v, ks, vs)
    plan = ops.SharedPrefixes([(64, [0, 1])], [65, 70], 2)
    for thing, names in ((cache, ("k", "v", "k_scale", "v_scale", "pointers", "pages", "n_kv_heads", "page_size", "head_dim", "device")),
                         (plan, ("plan", "pointers", "T", "group_heads", "tiles", "wide", "per_tile", "longest", "longest_prefix", "longest_rest", "device"))):
        for name in names:
            before = getattr(thing, name)
            with pytest.raises(AttributeError):
                setattr(thing, name, before)
            with pytest.raises(AttributeError):
                delattr(thing, name)
            assert getattr(thing, name) is before
    at = cache.pointers
    for t in (k, v, ks, vs):
        t.data = torch.empty(0, dtype=t.dtype, device="cuda")
    assert tuple(t.data_ptr() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)) == at
    torch.full((3, 2, 64, 64), 0, dtype=torch.uint8, device="cuda")         # (memory that was given back would be this one's)
    table = torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3)
    pos = torch.tensor([0, 130], dtype=torch.int32, device="cuda")
    rows = ops.kv_read_int8(cache, pos, torch.zeros(2, dtype=torch.int32, device="cuda"), table)
    assert (rows[0] == 3).all() and (rows[1] == 5).all()


@pytest.mark.parametrize("d", [64, 128, 32])
@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 300, 2 ** 30, 257])
def test_positions_beyond_the_table_are_reported_and_not_walked(ops, d, far):
    """A token whose position no page of the table can hold sees the positions that it can, or with a window none of them; the walk ends with the table."""
    pages = Pages(53, [256, 256], 2, d)
    cache, table, seq = pages.cache(ops), pages.table[:, :4].contiguous().cuda(), torch.arange(2, dtype=torch.int32).cuda()
    q = queries(54, 2, 4 * d).cuda()
    there, beyond = (torch.tensor([p, 99], dtype=torch.int32).cuda() for p in (255, far))
    assert take_error(ops) == 0
    for splits in (1, 3):
        want = ops.attention_decode_int8(q, cache, table, there, seq, 4, 0, 0.1, 256, splits=splits)
        assert take_error(ops) == 0
        got = ops.attention_decode_int8(q, cache, table, beyond, seq, 4, 0, 0.1, 256, splits=splits)
        assert take_error(ops) == 8 and torch.equal(got, want)
        for window in (1, -1):
            got = ops.attention_decode_int8(q, cache, table, beyond, seq, 4, window, 0.1, 256, splits=splits)
            assert take_error(ops) == 8 and (got[0] == 0).all() and (got[1] != 0).any()
    if d == 32:
        return
    cu, lens = torch.arange(3, dtype=torch.int32).cuda(), [torch.tensor([p + 1 if p + 1 < 2 ** 31 else p, 100], dtype=torch.int32).cuda() for p in (255, far)]
    want = ops.attention_prompts_int8(q, cache, table, cu, lens[0], 1, 4, 0, 0.1)
    assert take_error(ops) == 0
    got = ops.attention_prompts_int8(q, cache, table, cu, lens[1], 1, 4, 0, 0.1)
    assert take_error(ops) == 8 and torch.equal(got, want)
    got = ops.attention_prompts_int8(q, cache, table, cu, lens[1], 1, 4, 1, 0.1)
    assert take_error(ops) == 8 and (got[0] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("members", [2, 40])
@pytest.mark.parametrize("prefix", [2 ** 31 - 64, 2 ** 20])
def test_a_plan_that_goes_beyond_the_table_is_reported(ops, members, prefix):
    """Tiles of eight rows and of 256: the common positions that the table can name are walked, and the rest of a token's is empty."""
    pages = Pages(57, [256] * members, 2, 64)
    cache, table = pages.cache(ops), pages.table[:1, :4].expand(members, 4).contiguous().cuda()
    q, seq = queries(58, members, 4 * 64).cuda(), torch.arange(members, dtype=torch.int32).cuda()
    there, beyond = (torch.full((members,), p, dtype=torch.int32).cuda() for p in (255, prefix))
    made = [ops.SharedPrefixes([(p, list(range(members)))], [p + 1] * members, 2) for p in (192, prefix)]
    assert made[1].wide == (members == 40)
    want = ops.attention_decode_int8(q, cache, table, there, seq, 4, 0, 0.1, 256)
    assert take_error(ops) == 0
    got = ops.attention_decode_shared(q, cache, table, beyond, seq, made[1], 4, 0.1, prefix + 1, own_splits=2, pre_splits=4)
    assert take_error(ops) == 8
    assert (got.double() - want.double()).norm() <= 0.01 * want.double().norm()


CAPTURED_FIRST = """
import sys
import torch
from inferllm_b200.kernels import ops
kind, d, nh, n = sys.argv[1], 64, 4, 3
g = torch.Generator("cuda").manual_seed(1)
q = torch.randn((n, nh * d), generator=g, device="cuda").bfloat16()
qkv = torch.randn((n, (nh + 4) * d), generator=g, device="cuda").bfloat16()
table = torch.tensor([[0, 1], [0, 2], [0, 3]], dtype=torch.int32, device="cuda")
pos, seq = torch.tensor([70, 80, 127], dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
cu, lens, err = torch.arange(n + 1, dtype=torch.int32, device="cuda"), pos + 1, torch.zeros(1, dtype=torch.int32, device="cuda")
if kind != "wide":
    cache = ops.CacheInt8(*(torch.randint(0, 256, (4, 2, 64, d), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)),
                          *(torch.rand((4, 2, 64), generator=g, device="cuda") * 0.02 for _ in range(2)))
if kind in ("shared", "wide"):
    plan = ops.SharedPrefixes([(64, [0, 1, 2])], [71, 81, 128], nh // 2)
    pair = cache if kind == "shared" else tuple(torch.randn((4, 2, 64, d), generator=g, device="cuda").bfloat16() for _ in range(2))
call = {"decode": lambda: ops.attention_decode_int8(q, cache, table, pos, seq, nh, 0, 0.125, 128),
        "plain": lambda: ops.attention_decode_int8(q.float(), cache, table, pos, seq, nh, 0, 0.125, 128),
        "prompts": lambda: ops.attention_prompts_int8(q, cache, table, cu, lens, 1, nh, 0, 0.125),
        "rows": lambda: (ops.kv_write_int8(qkv, None, 0, pos, seq, table, cache, nh, err),) + ops.kv_read_int8(cache, pos, seq, table),
        "shared": lambda: ops.attention_decode_shared(q, pair, table, pos, seq, plan, nh, 0.125, 128),
        "wide": lambda: ops.attention_decode_shared(q, pair, table, pos, seq, plan, nh, 0.125, 128)}[kind]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
torch.cuda.synchronize()
want = call()
for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
    assert torch.equal(a, b) and (a != 0).any()
print("same")
"""


@pytest.mark.parametrize("kind", ["decode", "plain", "prompts", "rows", "shared", "wide"])
def test_a_call_that_is_captured_first_of_all(kind):
    """A process whose first call of the library goes into a graph: nothing is left to be made then."""
    out = subprocess.run([sys.executable, "-c", CAPTURED_FIRST, kind], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("same"), out.stderr[-2000:]


def test_scales_below_zero(ops):
    """A negative scale is computed where scores are scaled before their maximum is taken, and refused over common positions."""
    nh, nkv, d, n = 8, 2, 64, 20
    pages = Pages(61, [200 + i for i in range(n)], nkv, d, common=[(128, 0)] * n)
    cache, table = pages.cache(ops), pages.table.cuda()
    pos, seq = torch.tensor([199 + i for i in range(n)], dtype=torch.int32).cuda(), torch.arange(n, dtype=torch.int32).cuda()
    q = queries(62, n, nh * d)
    want, _ = expected(pages, q, [(i, 199 + i) for i in range(n)], nh, 0, -4.0, B8H)
    cu, lens = torch.arange(n + 1, dtype=torch.int32).cuda(), pos + 1
    for got in (ops.attention_decode_int8(q.cuda(), cache, table, pos, seq, nh, 0, -4.0, 256), ops.attention_prompts_int8(q.cuda(), cache, table, cu, lens, 1, nh, 0, -4.0)):
        assert torch.isfinite(got).all() and (got.double().cpu() - want).norm() <= 0.01 * want.norm()
    plan = ops.SharedPrefixes([(128, list(range(n)))], [200 + i for i in range(n)], nh // nkv)
    assert plan.wide
    for scale in (-0.1, float("nan")):
        with pytest.raises(KernelError, match="scale"):
            ops.attention_decode_shared(q.cuda(), cache, table, pos, seq, plan, nh, scale, 256)
    assert take_error(ops) == 0


def test_rows_further_apart_than_a_launch_can_say(ops):
    cache = ops.CacheInt8.empty(2, 2, 64, 64)
    q = torch.empty(2 ** 31 + 512, dtype=torch.bfloat16, device="cuda").as_strided((2, 512), (2 ** 31, 1))
    table, pos, seq = torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")
    with pytest.raises(KernelError, match="apart"):
        ops.attention_decode_int8(q, cache, table, pos, seq, 8, 0, 0.1, 64)


@pytest.mark.parametrize("nh, nkv, d, slices", [(4, 2, 64, 0), (32, 8, 128, 0), (3, 1, 24, 0), (2, 2, 256, 0), (32, 8, 128, 2)])
def test_values_fall_to_the_nearest_step(ops, nh, nkv, d, slices):
    """u = 128 + round(127 x / max |x|), halves to even, for rows as they come (bfloat16, not rotated), against whole numbers in 64 bits: 127 x is exact in float32 and a quotient of
    bfloat16 numbers that is no half is further from one than its rounding.  Rows hold their largest and its half, whose quotient is 63.5."""
    T = 500
    g = torch.Generator().manual_seed(nh * d)
    x = torch.randn((T, nh + 2 * nkv, d), generator=g) * torch.exp(4 * torch.randn((T, nh + 2 * nkv, 1), generator=g))
    x = x.bfloat16()
    top = x.float().abs().amax(-1, keepdim=True)
    x[:, :, 1:2] = (top / 2).bfloat16()
    x[:, :, 2:3] = (-top / 2).bfloat16()
    cache = ops.CacheInt8.empty(-(-T // 64), nkv, 64, d)
    pos, seq = torch.arange(T, dtype=torch.int32).cuda(), torch.zeros(T, dtype=torch.int32).cuda()
    table, err = torch.arange(cache.pages, dtype=torch.int32).cuda().view(1, -1), torch.zeros(1, dtype=torch.int32, device="cuda")
    qkv = x.reshape(T, -1).cuda()
    if slices:          # the first slice is the row, the others add nothing
        qkv = ops.SplitKPartials(torch.cat([qkv.float()[None], torch.zeros((slices - 1,) + qkv.shape, device="cuda")]).contiguous())
    ops.kv_write_int8(qkv, None, 0, pos, seq, table, cache, nh, err)
    for got, scale, rows in ((cache.k, cache.k_scale, x[:, nh:nh + nkv]), (cache.v, cache.v_scale, x[:, nh + nkv:])):
        a = rows.double().abs().amax(-1, keepdim=True)
        want = torch.round(127 * rows.double() / a) + 128
        u = got.cpu().transpose(1, 2).reshape(-1, nkv, d)[:T].double()
        assert torch.equal(u, want)
        s = scale.cpu().transpose(1, 2).reshape(-1, nkv)[:T]
        assert torch.equal(s, a[..., 0].float() / torch.full((T, nkv), 127.0))
    assert int(err.item()) == 0
