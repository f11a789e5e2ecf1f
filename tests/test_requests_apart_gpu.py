"""Requests of one batch that bring an adapter and sampling settings of their own, through the engine, the sampler and the entry
point (GPU).  An adapter's logits are held against the plain implementation with the adapter merged into its weights, with the
bounds of the other engine tests; adapters are as large as the weights they stand beside, so that a lost one is far outside them."""
import numpy as np
import plain_llama as plain
import pytest
import torch
from conftest import TINY, random_prompt
from test_sample_rows_gpu import choose
from util import assert_close

from inferllm_b200 import Engine, EngineError, EngineOptions, Model, ModelConfig, SamplingParams, StepItem
from inferllm_b200.kernels import ops
from inferllm_b200.sampling import Sampler, uniform_for

pytestmark = pytest.mark.gpu
ROLES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def factors(cfg, w, rank, seed, roles=ROLES, layers=None):
    """Factors beside these projections, as bfloat16 values, and the scale."""
    rng = np.random.default_rng(seed)
    out = {}
    for layer in range(cfg["num_hidden_layers"]) if layers is None else layers:
        for role in roles:
            name = f"model.layers.{layer}.{role}.weight"
            n, k = w[name].shape
            r = max(1, rank - seed % 3)
            a = torch.from_numpy(rng.standard_normal((r, k)).astype(np.float32) * k ** -0.5).bfloat16()
            b = torch.from_numpy(rng.standard_normal((n, r)).astype(np.float32) * 0.02 * (k / r) ** 0.5).bfloat16()
            out[name] = (a, b)
    return out, 0.5 + 0.25 * (seed % 4)


def merged(w, adapter):
    if adapter is None:
        return w
    out = dict(w)
    for name, (a, b) in adapter[0].items():
        out[name] = w[name] + adapter[1] * (b.double().numpy() @ a.double().numpy())
    return out


def engine(folder, dtype, **kw):
    return Engine.from_folder(folder, EngineOptions(dtype=dtype, max_tokens=kw.pop("max_tokens", 2048), max_batch=kw.pop("max_batch", 16), max_adapters=4,
                                                    adapter_rank=kw.pop("adapter_rank", 12), **kw))


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_adapters_of_a_batch(name, dtype, graphs, model_folders, plain_models):
    """Prompts of four requests in one step, then single tokens, each with its adapter, of other ranks, some on few projections."""
    cfg, w = plain_models[name]
    e = engine(model_folders[name], dtype, cuda_graphs=graphs)
    adapters = [factors(cfg, w, 12, 1), factors(cfg, w, 5, 2, ("self_attn.q_proj", "self_attn.v_proj")), factors(cfg, w, 12, 3, ROLES[3:], [1]), None]
    numbers = [e.add_adapter(*a) if a else -1 for a in adapters]
    assert numbers == [0, 1, 2, -1]
    prompts = [random_prompt(name, n, 60 + n) for n in (17, 40, 9, 23)]
    after = [random_prompt(name, 5, 90 + i) for i in range(4)]
    weights = [merged(w, a) for a in adapters]
    slots = [e.new_sequence() for _ in prompts]
    got = e.step([StepItem(s, p, list(range(len(p))), a) for s, p, a in zip(slots, prompts, numbers)]).cpu().numpy()
    at = 0
    for p, a, t in zip(prompts, weights, after):
        assert_close(got[at:at + len(p)], plain.forward(cfg, a, p), dtype, "prompt")
        at += len(p)
    want = [plain.forward(cfg, a, p + t)[len(p):] for p, a, t in zip(prompts, weights, after)]
    for j in range(5):          # the first single-token step runs as it is, the second is captured, the others replay it
        got = e.step([StepItem(s, [t[j]], [0], a) for s, t, a in zip(slots, after, numbers)]).cpu().numpy()
        for i in range(4):
            assert_close(got[i:i + 1], want[i][j:j + 1], dtype, f"token {j} of request {i}")
    e.check_device_errors()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_adapters_of_single_prompts(dtype, model_folders, plain_models):
    """Single prompts are padded and replayed from graphs: short and long ones (both forms of the product), first without, then
    with one adapter and another."""
    name = "C"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], dtype)
    adapters = [factors(cfg, w, 12, 4), factors(cfg, w, 3, 6)]
    numbers = [e.add_adapter(*a) for a in adapters]
    for length in (50, 250):
        p = random_prompt(name, length, length)
        for i in (None, 0, 1, 0, 1, None):
            slot = e.new_sequence()
            got = e.step([StepItem(slot, p, [length - 1], -1 if i is None else numbers[i])]).cpu().numpy()
            e.end_sequence(slot)
            assert_close(got, plain.forward(cfg, merged(w, None if i is None else adapters[i]), p)[-1:], dtype, f"{length} tokens, adapter {i}")


def test_many_sequences(model_folders, plain_models):
    """Single tokens of 140 sequences: more than the rows form takes, replayed from a graph with places for every adapter."""
    name = "A"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], "bfloat16", max_tokens=140 * 64, max_batch=140)
    adapters = [factors(cfg, w, 12, s) for s in (1, 2, 3, 4)]
    for a in adapters:
        e.add_adapter(*a)
    p = random_prompt(name, 4, 4)
    slots = [e.new_sequence() for _ in range(140)]
    for s in range(0, 140, 35):
        e.step([StepItem(x, p[:1], [], -1 if x % 5 == 4 else x % 5) for x in slots[s:s + 35]])
    want = [plain.forward(cfg, merged(w, a), p) for a in adapters + [None]]
    for j in (1, 2, 3):
        got = e.step([StepItem(x, [p[j]], [0], -1 if x % 5 == 4 else x % 5) for x in slots]).cpu().numpy()
        for i, x in enumerate(slots):
            assert_close(got[i:i + 1], want[x % 5][j:j + 1], "bfloat16", f"sequence {x}, token {j}")


def test_float32_sequences_without_an_adapter_keep_their_bits(model_folders, plain_models):
    name = "C"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], "float32")
    a = e.add_adapter(*factors(cfg, w, 12, 1))
    p, q = random_prompt(name, 30, 1), random_prompt(name, 12, 2)

    def run(adapter):
        s, t = e.new_sequence(), e.new_sequence()
        out = [e.step([StepItem(s, p, [29], adapter), StepItem(t, q, [11])])[1]]
        out += [e.step([StepItem(s, [5], [0], adapter), StepItem(t, [j], [0])])[1] for j in range(3)]
        e.end_sequence(s)
        e.end_sequence(t)
        return torch.stack(out)

    assert torch.equal(run(-1), run(a))


def test_adapters_come_and_go(model_folders, plain_models):
    name = "A"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], "float32")
    p = random_prompt(name, 11, 3)

    def logits(adapter):
        s = e.new_sequence()
        out = e.step([StepItem(s, p, [10], adapter)]).cpu().numpy()
        e.end_sequence(s)
        return out

    first, second = factors(cfg, w, 12, 1), factors(cfg, w, 2, 2, ROLES[:1])
    assert [e.add_adapter(*first) for _ in range(4)] == [0, 1, 2, 3]
    with pytest.raises(EngineError):
        e.add_adapter(*first)
    e.remove_adapter(2)
    with pytest.raises(EngineError):
        logits(2)
    with pytest.raises(EngineError):
        e.remove_adapter(2)
    assert e.add_adapter(*second) == 2
    assert_close(logits(2), plain.forward(cfg, merged(w, second), p)[-1:], "float32", "the second in the first's place")
    assert_close(logits(3), plain.forward(cfg, merged(w, first), p)[-1:], "float32", "the first")


def test_refusals(model_folders, plain_models):
    name = "A"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], "bfloat16")
    good, scale = factors(cfg, w, 4, 3)
    q = "model.layers.0.self_attn.q_proj.weight"
    a, b = good[q]
    assert set(e.adapted()) == {f"model.layers.{i}.{r}.weight" for i in range(2) for r in ROLES} and e.adapted()[q] == w[q].shape
    for bad in ({}, {"model.norm.weight": (a, b)}, {q: (a[:, :-1], b)}, {q: (a, b[:-1])}, {q: (a[:2], b)}, {q: (torch.zeros(13, 64), torch.zeros(64, 13))},
                {q: (torch.zeros(0, 64), torch.zeros(64, 0))}, {q: (a * float("inf"), b)}, {q: (a, b * float("nan"))}):
        with pytest.raises(EngineError):
            e.add_adapter(bad, scale)
    with pytest.raises(EngineError):
        e.add_adapter(good, float("nan"))
    s = e.new_sequence()
    for number in (0, -2, 4):
        with pytest.raises(EngineError):
            e.step([StepItem(s, [1, 2], [1], number)])
    with pytest.raises(EngineError):
        Engine.from_folder(model_folders[name], EngineOptions(max_adapters=2, adapter_rank=86))
    plain_engine = Engine.from_folder(model_folders[name], EngineOptions(max_tokens=256))
    with pytest.raises(EngineError):
        plain_engine.add_adapter(good, scale)


# ---- settings per request


def penalised(logits, history, penalty, n):
    out = np.asarray(logits, np.float32).copy()
    for t in set(history[-n:]) if n else ():
        out[t] = out[t] * np.float32(penalty) if out[t] < 0 else out[t] / np.float32(penalty)
    return out


EACH = [SamplingParams(), SamplingParams(temp=1.0, seed=3), SamplingParams(temp=0.7, top_k=20, top_p=0.9, seed=4), SamplingParams(temp=1.3, min_p=0.2, seed=5),
        SamplingParams(temp=0.9, top_p=0.5, repeat_penalty=1.5, repeat_last_n=6, seed=6), SamplingParams(repeat_penalty=1.7, repeat_last_n=6, seed=7)]


def expect(logits, p, request, step, history):
    f = np.float32
    l = penalised(logits, history, p.repeat_penalty, p.repeat_last_n) if p.repeat_penalty != 1.0 else logits
    return choose(l, float(f(uniform_for(p.seed, request, step))), float(f(p.temp)), p.top_k, float(f(p.top_p)), float(f(p.min_p)))


def test_settings_of_their_own(model_folders):
    e = Engine.from_folder(model_folders["A"], EngineOptions(max_tokens=512))
    g = torch.Generator("cuda").manual_seed(1)
    sampler = Sampler(e, EACH)
    rng = np.random.default_rng(2)
    histories = [rng.integers(0, 300, 9).tolist() for _ in EACH]
    for step in range(4):
        logits = torch.randn((len(EACH), 300), generator=g, device="cuda") * 3
        kept = logits.clone()
        order = [3, 0, 5, 1, 4, 2]
        got = sampler.choose(logits[order].contiguous(), order, [step] * 6, [histories[r] for r in order]).tolist()
        assert torch.equal(logits, kept)
        assert got == [expect(logits[r].cpu().numpy(), EACH[r], r, step, histories[r]) for r in order]
        for r, t in zip(order, got):
            histories[r].append(t)


def test_min_p_for_all(model_folders):
    e = Engine.from_folder(model_folders["A"], EngineOptions(max_tokens=512))
    logits = torch.randn((7, 300), generator=torch.Generator("cuda").manual_seed(3), device="cuda") * 2
    p = SamplingParams(temp=1.1, top_k=50, min_p=0.1, seed=9)
    got = Sampler(e, p).choose(logits, list(range(7)), [2] * 7).tolist()
    assert got == [expect(logits[r].cpu().numpy(), p, r, 2, []) for r in range(7)]


def test_sampler_refusals(model_folders):
    e = Engine.from_folder(model_folders["A"], EngineOptions(max_tokens=512))
    for bad in ([], [SamplingParams(min_p=1.5)], [SamplingParams(min_p=-0.1)], [SamplingParams(repeat_penalty=1.1, repeat_last_n=5), SamplingParams(repeat_penalty=1.1, repeat_last_n=6)]):
        with pytest.raises(ValueError):
            Sampler(e, bad)
    with pytest.raises(ValueError):
        Sampler(e, [SamplingParams()]).choose(torch.zeros((2, 10), device="cuda"), [0, 1], [0, 0])


# ---- both together


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation(dtype, model_folders, plain_models):
    """Requests with adapters and settings of their own in one batch give what each gives by itself (float32: to the token), and
    greedy ones what the plain implementation gives with the adapter merged."""
    name = "B"
    cfg, w = plain_models[name]
    m = Model(ModelConfig(compt_type=dtype, nr_ctx=TINY[name]["max_position_embeddings"], max_tokens=1024, max_adapters=3, adapter_rank=8))
    m.load(model_folders[name])
    m.init(top_k=0, top_p=1.0, temp=0.0, repeat_penalty=1.0, repeat_last_n=0, seed=0, end_token=-1)
    adapters = [factors(cfg, w, 8, 3), factors(cfg, w, 4, 6, ROLES[4:])]
    numbers = [m.engine.add_adapter(*a) for a in adapters]
    prompts = [random_prompt(name, n, 300 + n) for n in (12, 5, 31, 8, 20)]
    which, n_new = [numbers[0], -1, numbers[1], numbers[0], -1], 7
    greedy = m.generate(prompts, max_new_tokens=n_new, stop_ids=[], adapters=which).tokens
    want = [plain.greedy_generate(cfg, merged(w, adapters[a] if a >= 0 else None), p, n_new) for p, a in zip(prompts, which)]
    if dtype == "float32":
        assert greedy == want
    else:                       # bfloat16 may turn a near-tie the other way; the first tokens must agree
        assert all(g[0] == v[0] for g, v in zip(greedy, want)) and sum(g == v for g, v in zip(greedy, want)) >= 4
    each = [SamplingParams(temp=0.8, seed=11), SamplingParams(), SamplingParams(temp=1.0, top_k=30, min_p=0.05, seed=12),
            SamplingParams(temp=1.2, top_p=0.8, repeat_penalty=1.3, repeat_last_n=8, seed=13), SamplingParams(repeat_penalty=1.3, repeat_last_n=8)]
    out = m.generate(prompts, max_new_tokens=n_new, stop_ids=[], adapters=which, sampling=each).tokens
    assert out[1] == greedy[1] and [len(t) for t in out] == [n_new] * 5
    again = m.generate(prompts, max_new_tokens=n_new, stop_ids=[], adapters=which, sampling=each).tokens
    assert out == again
    if dtype == "float32":
        for i in (0, 2, 3):     # (request numbers key the random numbers: the others stand in front as one-token prompts)
            filler = [[1]] * i
            alone = m.generate(filler + [prompts[i]], max_new_tokens=n_new, stop_ids=[], adapters=[-1] * i + [which[i]], sampling=each[:i + 1]).tokens
            assert alone[i] == out[i]
    with pytest.raises(ValueError):
        m.generate(prompts, sampling=each[:2])
    with pytest.raises(ValueError):
        m.generate(prompts, adapters=[0])


def test_the_operators_one_behind_another():
    """A head's product with adapters, its float32 rows straight into the choice of a token, captured and replayed."""
    g = torch.Generator("cuda").manual_seed(4)
    T, K, V = 24, 256, 5000
    x, w = torch.randn((T, K), generator=g, device="cuda").bfloat16(), (torch.randn((V, K), generator=g, device="cuda") * 0.2).bfloat16()
    ad = ops.Adapters(3, 16, V, K)
    parts = [(torch.randn((16, K), generator=g, device="cuda") / 16, torch.randn((V, 16), generator=g, device="cuda")) for _ in range(3)]
    for i, (a, b) in enumerate(parts):
        ad.put(i, a, b, 0.7)
    index = [t % 4 - 1 for t in range(T)]
    rows, u = ops.AdapterRows(index, ad.ranks), torch.rand(T, generator=g, device="cuda")
    temp, k, p = torch.full((T,), 0.8, device="cuda"), torch.full((T,), 30, dtype=torch.int32, device="cuda"), torch.full((T,), 0.9, device="cuda")

    def both():
        logits = ops.linear_adapters(x, w, ad, rows, torch.float32)
        return logits, ops.sample_rows(logits, u, temp, k, p)

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, tokens = both()
    for seed in range(3):
        x.copy_(torch.randn((T, K), generator=g, device="cuda"))
        graph.replay()
        l, t = both()
        assert torch.equal(l, logits) and torch.equal(t, tokens)
        host = logits.double().cpu().numpy()
        assert tokens.tolist() == [choose(host[i], float(u[i]), float(np.float32(0.8)), 30, float(np.float32(0.9))) for i in range(T)]


@pytest.mark.parametrize("max_adapters", [4, 40])
def test_captured_steps_of_72_sequences(max_adapters, model_folders, plain_models):
    """Room for few adapters (tiles of tokens) or for many (token by token, whatever the step names)."""
    name, n = "A", 72
    cfg, w = plain_models[name]
    e = Engine.from_folder(model_folders[name], EngineOptions(dtype="bfloat16", max_tokens=n * 64, max_batch=n, max_adapters=max_adapters, adapter_rank=12))
    adapters = [factors(cfg, w, 12, s) for s in (1, 2, 3)]
    for a in adapters:
        e.add_adapter(*a)
    p = random_prompt(name, 5, 4)
    slots = [e.new_sequence() for _ in range(n)]
    for s in range(0, n, 36):
        e.step([StepItem(x, p[:1], [], -1 if x % 4 == 3 else x % 4) for x in slots[s:s + 36]])
    want = [plain.forward(cfg, merged(w, a), p) for a in adapters + [None]]
    for j in (1, 2, 3, 4):
        got = e.step([StepItem(x, [p[j]], [0], -1 if x % 4 == 3 else x % 4) for x in slots]).cpu().numpy()
        for i, x in enumerate(slots):
            assert_close(got[i:i + 1], want[x % 4][j:j + 1], "bfloat16", f"sequence {x}, token {j}")


def test_cache_sized_from_the_memory_that_adapters_leave(model_folders):
    """Where the cache takes a share of the free memory, it is of what the room for adapters leaves."""
    import gc

    def made(**kw):
        """Pages of the cache, and bytes of device memory that the engine took."""
        gc.collect()
        torch.cuda.empty_cache()
        free = torch.cuda.mem_get_info()[0]
        e = Engine.from_folder(model_folders["C"], EngineOptions(dtype="bfloat16", max_batch=4, adapter_rank=85, **kw))
        out = e.limits().num_pages, free - torch.cuda.mem_get_info()[0]
        del e
        return out

    made(max_tokens=64)
    room = made(max_tokens=64, max_adapters=4096)[1] - made(max_tokens=64)[1]
    page = 64 * 2 * 2 * 2 * 128 * 2         # tokens, layers, keys and values, heads, channels, bytes
    assert room > 10e9
    without, beside = made(max_tokens=None, mem_fraction=0.05)[0], made(max_tokens=None, mem_fraction=0.05, max_adapters=4096)[0]
    assert abs((without - beside) * page - 0.05 * room) < 0.1 * 0.05 * room


def test_requests_that_end_at_different_times(model_folders):
    """Settings, windows of last tokens and adapters of their own while requests leave the batch one after another, against one
    request at a time with its choices written out (float32: the logits do not depend on the batch)."""
    name, n_new = "B", 12
    m = Model(ModelConfig(compt_type="float32", nr_ctx=TINY[name]["max_position_embeddings"], max_tokens=2048, max_adapters=3, adapter_rank=8))
    m.load(model_folders[name])
    m.init(top_k=0, top_p=1.0, temp=0.0, repeat_penalty=1.0, repeat_last_n=0, seed=0, end_token=-1)
    import plain_llama
    cfg, w = plain_llama.load_weights(model_folders[name])
    numbers = [m.engine.add_adapter(*factors(cfg, w, 8, s)) for s in (3, 6)]
    prompts = [random_prompt(name, n, 400 + n) for n in (9, 30, 4, 17, 22, 6, 13)]
    which = [numbers[i % 3] if i % 3 < 2 else -1 for i in range(7)]
    each = [SamplingParams(temp=(0.0, 0.8, 1.2, 1.0)[i % 4], top_k=(0, 30)[i % 2], top_p=(1.0, 0.9, 0.7)[i % 3], min_p=(0.0, 0.03)[i // 2 % 2], seed=20 + i,
                           repeat_penalty=(1.4, 1.0, 2.0, 0.7)[(i + 1) % 4], repeat_last_n=(5, 0)[(i + 1) % 4 == 1]) for i in range(7)]

    def alone(r, stop):
        slot, history, out = m.engine.new_sequence(), list(prompts[r]), []
        feed = history
        for step in range(n_new):
            logits = m.engine.step([StepItem(slot, feed, [len(feed) - 1], which[r])])[0].cpu().numpy()
            out.append(expect(logits, each[r], r, step, history))
            history, feed = history + out[-1:], out[-1:]
            if out[-1] in stop:
                break
        m.engine.end_sequence(slot)
        return out

    free = m.generate(prompts, max_new_tokens=n_new, stop_ids=[], sampling=each, adapters=which)
    assert free.tokens == [alone(r, ()) for r in range(7)]
    stop = {free.tokens[r][at] for r, at in ((0, 2), (3, 0), (4, 5), (6, 8), (1, 3))}
    got = m.generate(prompts, max_new_tokens=n_new, stop_ids=sorted(stop), sampling=each, adapters=which)
    assert got.tokens == [alone(r, stop) for r in range(7)]
    assert len({len(t) for t in got.tokens}) >= 4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("max_adapters", [30, 64])
def test_many_sequences_with_many_adapters(max_adapters, dtype, model_folders, plain_models):
    """Single tokens of 150 sequences with 30 adapters among them, then of ever fewer of these."""
    name, n, used = "A", 150, 30
    cfg, w = plain_models[name]
    e = Engine.from_folder(model_folders[name], EngineOptions(dtype=dtype, max_tokens=n * 64, max_batch=n, max_adapters=max_adapters, adapter_rank=12))
    adapters = [factors(cfg, w, 12, s) for s in range(used)]
    for a in adapters:
        e.add_adapter(*a)
    p = random_prompt(name, 9, 4)
    which = [(x * 7) % (used + 1) - 1 for x in range(n)]
    want = [plain.forward(cfg, merged(w, a), p) for a in adapters + [None]]
    slots = [e.new_sequence() for _ in range(n)]
    for s in range(0, n, 50):
        e.step([StepItem(x, p[:1], [], which[x]) for x in slots[s:s + 50]])
    for j, live in ((1, 150), (2, 150), (3, 150), (4, 130), (5, 120), (6, 61), (7, 60), (8, 2)):
        got = e.step([StepItem(x, [p[j]], [0], which[x]) for x in slots[:live]]).cpu().numpy()
        for i in range(live):
            assert_close(got[i:i + 1], want[which[i]][j:j + 1], dtype, f"sequence {i}, token {j}")
    e.check_device_errors()
