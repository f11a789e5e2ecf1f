"""The engine with a cache of eight-bit rows, and sequences that share their first positions (GPU).

The plain implementation is given the same rounding of keys and values.  A value that lies on the border between two steps may
fall to either side in the engine, which moves it by 1/127 of its row's largest: less than what rounding every activation to bfloat16 does, whose bounds
therefore serve the float32 mode here too."""
import os
import subprocess
from dataclasses import dataclass

import numpy as np
import plain_llama as plain
import pytest
import torch
from conftest import ROOT, TINY, random_prompt
from util import assert_close

from inferllm_b200 import CacheError, Engine, EngineError, EngineOptions, Model, ModelConfig, StepItem, write_random_model
from inferllm_b200.config import ArchConfig, LayerSpec, ModelSpec, PartSpec, ScheduleEntry, register_architecture, unregister_architecture
from inferllm_b200.kernels import ops
from inferllm_b200.parts import PositionEncoding, register_position, unregister_part

pytestmark = pytest.mark.gpu


def eight_bits(x):
    s = np.abs(x).max(-1, keepdims=True) / 127
    return np.rint(x / np.where(s > 0, s, 1)) * s


@pytest.fixture
def rounded(monkeypatch):
    """The plain implementation over keys and values of eight bits."""
    scores, values = plain.attention_scores, plain.weighted_values
    monkeypatch.setattr(plain, "attention_scores", lambda q, k, *a: scores(q, eight_bits(k), *a))
    monkeypatch.setattr(plain, "weighted_values", lambda p, v, *a: values(p, eight_bits(v), *a))


def engine(folder, dtype="bfloat16", cache="int8", **kw):
    return Engine.from_folder(folder, EngineOptions(dtype=dtype, cache_dtype=cache, max_tokens=kw.pop("max_tokens", 4096), max_batch=kw.pop("max_batch", 16), **kw))


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_logits(name, dtype, graphs, model_folders, plain_models, rounded):
    """Three prompts in one step, then single tokens (the second such step is captured, the others replay it)."""
    cfg, w = plain_models[name]
    e = engine(model_folders[name], dtype, cuda_graphs=graphs, poison_freed_pages=True)
    prompts, after = [random_prompt(name, n, 30 + n) for n in (17, 70, 9)], [random_prompt(name, 5, 40 + i) for i in range(3)]
    slots = [e.new_sequence() for _ in prompts]
    got, at = e.step([StepItem(s, p, list(range(len(p)))) for s, p in zip(slots, prompts)]).cpu().numpy(), 0
    for p in prompts:
        assert_close(got[at:at + len(p)], plain.forward(cfg, w, p), "bfloat16", "prompt")
        at += len(p)
    want = [plain.forward(cfg, w, p + t)[len(p):] for p, t in zip(prompts, after)]
    for j in range(5):
        got = e.step([StepItem(s, [t[j]], [0]) for s, t in zip(slots, after)]).cpu().numpy()
        for i in range(3):
            assert_close(got[i:i + 1], want[i][j:j + 1], "bfloat16", f"token {j} of request {i}")
    e.check_device_errors()
    # a page that comes back from the pool is another sequence's no more
    for s in slots:
        e.end_sequence(s)
    p = random_prompt(name, 33, 77)
    assert_close(e.step([StepItem(e.new_sequence(), p, list(range(33)))]).cpu().numpy(), plain.forward(cfg, w, p), "bfloat16", "reused pages")
    e.check_device_errors()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "C", "D"])
def test_a_prompt_in_pieces(name, dtype, model_folders):
    """At once, in pieces and token by token: the same rows end up in the cache.  Single prompts are padded and replayed from graphs too."""
    e = engine(model_folders[name], dtype)
    p = random_prompt(name, 130, 5)
    for _ in range(3):
        whole = e.step([StepItem(s := e.new_sequence(), p, [129])])
        e.end_sequence(s)
    s = e.new_sequence()
    for a, b in ((0, 50), (50, 51), (51, 129)):
        e.step([StepItem(s, p[a:b], [])])
    pieces = e.step([StepItem(s, p[129:], [0])])
    s = e.new_sequence()
    for t in p[:-1]:
        e.step([StepItem(s, [t], [])])
    singles = e.step([StepItem(s, p[-1:], [0])])
    e.check_device_errors()
    for other in (pieces, singles):
        assert_close(other.cpu().numpy(), whole.cpu().numpy(), "bfloat16")


HIDDEN, HEADS, KV_HEADS, SIZE, WORDS, WINDOW, BASE = 96, 4, 2, 64, 90, 70, 1e4


@register_position("pairs_of_a_test")
class Pairs(PositionEncoding):
    """An encoding of its own, which writes rows of the activations' type: its layer's entry stays wide."""

    def encode_and_store(self, qkv, geometry, ctx, kv):
        nh, nkv, d = geometry
        ops.rope_kv_write(qkv, None, 0, ctx.token_pos, ctx.token_seq, kv.block_table, kv.k, kv.v, nh, nkv, d, kv.page_size, True, ctx.err)
        return qkv


@dataclass
class ManyKinds(ArchConfig):
    """Attention with a window and without, a layer that reads another's entry and, `own`, one that cannot keep eight bits."""
    own: bool = False

    @classmethod
    def from_dict(cls, d):
        return cls(own=d["own"])

    def to_dict(self):
        return {"architectures": ["ManyKindsForCausalLM"], "own": self.own}

    def model_spec(self):
        norm = PartSpec("rmsnorm", {"size": HIDDEN, "eps": 1e-5})
        shape = {"hidden_size": HIDDEN, "n_heads": HEADS, "n_kv_heads": KV_HEADS, "head_dim": SIZE}
        half = PartSpec("rope_half", {"head_dim": SIZE, "theta": BASE, "max_positions": 512})
        mixers = [PartSpec("attention", dict(shape, window=w, position=p)) for w, p in
                  [(None, half), (WINDOW, half), (None, half), (None, PartSpec("pairs_of_a_test", {}))][:4 if self.own else 3]]
        ffn = PartSpec("gated_mlp", {"hidden_size": HIDDEN, "intermediate_size": 128})
        layers = [LayerSpec("prenorm", m, ffn, {"norm1": norm, "norm2": norm}, f"blocks.{i}.", {"mixer": "mixer.", "ffn": "ffn.", "norm1": "ln1.", "norm2": "ln2."})
                  for i, m in enumerate(mixers)]
        schedule = [ScheduleEntry(0, 0), ScheduleEntry(1, 1), ScheduleEntry(2, 0, writes=False)] + ([ScheduleEntry(3, 2)] if self.own else [])
        return ModelSpec(HIDDEN, WORDS, layers, schedule, PartSpec("embedding", {"name": "emb.", "vocab_size": WORDS, "hidden_size": HIDDEN}),
                         PartSpec("rmsnorm", {"name": "ln_f.", "size": HIDDEN, "eps": 1e-5}),
                         PartSpec("lm_head", {"name": "head.", "tied": True, "vocab_size": WORDS, "hidden_size": HIDDEN}), 512, None, [])


def plain_many(w, ids, own):
    pos, x, kept = np.arange(len(ids)), plain.embed(ids, w["emb.weight"]), {}
    for layer, entry in [(0, 0), (1, 1), (2, 0), (3, 2)][:4 if own else 3]:
        p = f"blocks.{layer}."
        h = plain.rms_norm(x, w[p + "ln1.weight"], 1e-5)
        weights = [w[p + f"mixer.{n}_proj.weight"] for n in "qkvo"]
        if layer == 3:
            q, k, v = (plain.linear(h, m).reshape(len(ids), -1, SIZE) for m in weights[:3])
            s = plain.scale_and_mask(plain.attention_scores(q, k, HEADS, KV_HEADS), SIZE ** -0.5)
            a = plain.linear(plain.weighted_values(plain.softmax_rows(s), v, HEADS, KV_HEADS), weights[3])
        else:
            shape = pos, HEADS, KV_HEADS, SIZE, BASE
            if layer < 2:
                kept[entry] = tuple(eight_bits(t) for t in plain.self_attention(h, *weights, *shape)[1])
            a, _ = plain.self_attention(h, *weights, *shape, window=WINDOW if layer == 1 else None, kv_override=kept[entry])
        x = x + a
        h = plain.rms_norm(x, w[p + "ln2.weight"], 1e-5)
        x = x + plain.swiglu_ffn(h, *(w[p + f"ffn.{n}_proj.weight"] for n in ("gate", "up", "down")))
    return plain.linear(plain.rms_norm(x, w["ln_f.weight"], 1e-5), w["emb.weight"])


@pytest.fixture(scope="module", params=[False, True])
def many_kinds(request, tmp_path_factory):
    register_architecture("ManyKindsForCausalLM", ManyKinds)
    d = str(tmp_path_factory.mktemp("many"))
    write_random_model(ManyKinds(own=request.param), d, seed=5, dtype=torch.bfloat16)
    yield d, request.param
    unregister_architecture("ManyKindsForCausalLM")
    if request.param:
        unregister_part("position", "pairs_of_a_test")


@pytest.mark.parametrize("dtype, page", [("float32", 16), ("bfloat16", 64), ("bfloat16", 16)])
def test_windows_and_entries_that_layers_share(many_kinds, dtype, page):
    """Past the window, where pages go back (and are poisoned) while the sequences grow; entries in eight bits beside one that stays wide."""
    folder, own = many_kinds
    _, w = plain.load_weights(folder)
    e = engine(folder, dtype, page_size=page, poison_freed_pages=True)
    assert [g.get("k_scale") is not None for g in e.cache.stats()["paged"]].count(True) == 2
    rng = np.random.default_rng(7)
    texts = [rng.integers(0, WORDS, n).tolist() for n in (230, 60, 150)]
    first = [200, 30, 1]
    slots = [e.new_sequence() for _ in texts]
    refs = [plain_many(w, t, own) for t in texts]
    got, at = e.step([StepItem(s, t[:n], list(range(n))) for s, t, n in zip(slots, texts, first)]).cpu().numpy(), 0
    for r, n in zip(refs, first):
        assert_close(got[at:at + n], r[:n], "bfloat16", "prompt")
        at += n
    for j in range(30):
        got = e.step([StepItem(s, [t[n + j]], [0]) for s, t, n in zip(slots, texts, first)]).cpu().numpy()
        for i in range(3):
            assert_close(got[i:i + 1], refs[i][first[i] + j:first[i] + j + 1], "bfloat16", f"token {j} of request {i}")
    # the last one's next tokens in one step, on top of what is there
    got = e.step([StepItem(slots[2], texts[2][31:], list(range(119)))]).cpu().numpy()
    assert_close(got, refs[2][31:], "bfloat16", "a longer piece")
    e.check_device_errors()
    with pytest.raises(CacheError):
        e.fork_sequence(slots[0], 64)
    for s in slots:
        e.end_sequence(s)
    e.cache.check()


def test_what_lies_in_the_cache(model_folders, plain_models):
    """The first layer's rows: the plain implementation's keys and values in eight bits."""
    name = "C"
    cfg, w = plain_models[name]
    e = engine(model_folders[name], "float32")
    p = random_prompt(name, 100, 3)
    s = e.new_sequence()
    e.step([StepItem(s, p, [99])])
    k, v, ks, vs = e.cache_tensors(0)
    assert k.dtype == torch.uint8 and ks.shape == k.shape[:-1]
    layer = ops.CacheInt8(k[0], v[0], ks[0], vs[0])
    pages = e.cache.pages_of(0, s)
    table = torch.tensor([[pages[i] for i in range(2)]], dtype=torch.int32).cuda()
    got = ops.kv_read_int8(layer, torch.arange(100, dtype=torch.int32).cuda(), torch.zeros(100, dtype=torch.int32).cuda(), table, torch.float32)
    h = plain.rms_norm(plain.embed(p, w["model.embed_tokens.weight"]), w["model.layers.0.input_layernorm.weight"], cfg["rms_norm_eps"])
    shape = (100, cfg["num_key_value_heads"], cfg["head_dim"])
    want_k = plain.rope_rotate_half(plain.linear(h, w["model.layers.0.self_attn.k_proj.weight"]).reshape(shape), np.arange(100), cfg["rope_theta"])
    want_v = plain.linear(h, w["model.layers.0.self_attn.v_proj.weight"]).reshape(shape)
    for g, x in zip(got, (want_k, want_v)):
        # half a step, and float32's way to the row (a few hundred roundings of 2^-24)
        step = np.abs(x).max(-1, keepdims=True) / 127
        assert (np.abs(g.cpu().numpy() - x) <= step * (0.5 + 0.01)).all()


# ---------------------------------------------------------------- shared positions

SHARED = {"C": (640, 512), "D": (400, 320)}


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("cache", ["auto", "int8"])
@pytest.mark.parametrize("name", ["C", "D"])
@pytest.mark.parametrize("n", [4, 14, 100])
def test_forks_answer_as_if_they_were_alone(name, cache, graphs, n, model_folders, plain_models, monkeypatch, request):
    """Sequences that share a prefix with the one that made it, each with tokens of its own, beside one that shares nothing: enough of them that their
    steps walk the prefix once (in tiles of 8 and 256 rows)."""
    if cache == "int8":
        request.getfixturevalue("rounded")
    cfg, w = plain_models[name]
    e = engine(model_folders[name], cache=cache, cuda_graphs=graphs, max_tokens=8192 if n < 100 else 32768, max_batch=n + 3, shared_prefix_bytes=0)
    prompt = random_prompt(name, SHARED[name][0], 11)
    common = SHARED[name][1]
    slots = [e.new_sequence()]
    e.step([StepItem(slots[0], prompt, [])])
    slots += [e.fork_sequence(slots[0], common) for _ in range(n - 1)]
    texts = [prompt] + [prompt[:common] + random_prompt(name, 3 + i % 40, 200 + i) for i in range(n - 1)]
    lone = random_prompt(name, 21, 12)
    slots.append(e.new_sequence())
    texts.append(lone)
    # the forks' own tokens as short prompts
    items = [StepItem(s, t[common:], [len(t) - common - 1]) for s, t in zip(slots[1:n], texts[1:n])] + [StepItem(slots[n], lone, [20])]
    got = e.step(items).cpu().numpy()
    some = [1, n - 1, n]
    for i in some:
        assert_close(got[i - 1:i], plain.forward(cfg, w, texts[i])[-1:], "bfloat16", f"prompt of {i}")
    for j in range(4):
        tokens = [random_prompt(name, 1, 300 + 20 * j + i) for i in range(n + 1)]
        texts = [t + x for t, x in zip(texts, tokens)]
        got = e.step([StepItem(s, x, [0]) for s, x in zip(slots, tokens)]).cpu().numpy()
        for i in [0] + some:
            assert_close(got[i:i + 1], plain.forward(cfg, w, texts[i])[-1:], "bfloat16", f"token {j} of {i}")
    e.check_device_errors()
    # the sequence that made the prefix ends first, in a step of other sizes
    e.end_sequence(slots[0])
    tokens = [random_prompt(name, 1, 500 + i) for i in range(n + 1)]
    texts = [t + x for t, x in zip(texts, tokens)]
    order = list(range(n, 0, -1))
    got = e.step([StepItem(slots[i], tokens[i], [0]) for i in order]).cpu().numpy()
    for i in some:
        at = order.index(i)
        assert_close(got[at:at + 1], plain.forward(cfg, w, texts[i])[-1:], "bfloat16", f"after the end, {i}")
    e.check_device_errors()
    for s in slots[1:]:
        e.end_sequence(s)
    e.cache.check()
    assert e.cache.pages_free() == [e.limits().num_pages]


def test_common_positions_are_walked_once_where_that_saves_enough(model_folders):
    """A narrow tile adds the kernel that joins the shares, a wide one its own kernel too; a step that would save less is as before."""
    launches = {}
    for least in (0, 256 * 2 * 4 * 128 * 128, 2 ** 63 - 1, -1):
        e = engine(model_folders["C"], cache="int8", cuda_graphs=False, max_batch=16, shared_prefix_bytes=least)
        a = e.new_sequence()
        e.step([StepItem(a, random_prompt("C", 256, 1), [])])
        slots = [a] + [e.fork_sequence(a, 256) for _ in range(2)]
        items = [StepItem(s, random_prompt("C", 1, 2 + i), [0]) for i, s in enumerate(slots)]
        e.step(items)
        before = ops.launch_count()
        e.step(items)
        launches[least] = ops.launch_count() - before
        e.check_device_errors()
    few, some, none, rule = launches.values()
    assert few > some == none == rule


@pytest.mark.parametrize("name, dtype, cache", [("A", "float32", "int8"), ("B", "float32", "auto"), ("B", "bfloat16", "int8"), ("D", "float32", "int8")])
def test_forks_on_the_plain_kernels(name, dtype, cache, model_folders):
    """Sizes and types that read a shared prefix for every sequence: a fork answers as the same tokens in a sequence of their own."""
    e = engine(model_folders[name], dtype, cache=cache, page_size=16)
    prompt, tail = random_prompt(name, 70, 1), random_prompt(name, 6, 2)
    a, b = e.new_sequence(), e.new_sequence()
    e.step([StepItem(a, prompt, [])])
    e.step([StepItem(b, prompt[:64], [])])
    c = e.fork_sequence(a, 64)
    for t in tail:
        got = e.step([StepItem(b, [t], [0]), StepItem(c, [t], [0])]).cpu()
        assert_close(got[:1].numpy(), got[1:].numpy(), dtype)
    e.check_device_errors()


def test_generate_runs_common_positions_once(model_folders):
    """The same tokens with and without, in float32, where a row's result does not depend on what else is in the step; and fewer tokens to run."""
    name = "C"
    head = random_prompt(name, 150, 1)
    prompts = [head + random_prompt(name, 2 + i, 50 + i) for i in range(5)] + [head[:149]]
    results = []
    for share in (False, True):
        m = Model(ModelConfig(compt_type="float32", nr_ctx=512, max_tokens=4096, share_prefixes=share))
        m.load(model_folders[name])
        m.init(top_k=40, top_p=0.95, temp=0.0, repeat_penalty=1.0, repeat_last_n=64, seed=1, end_token=2)
        results.append(m.generate(prompts, max_new_tokens=8, stop_ids=[]).tokens)
        m.engine.check_device_errors()
        assert m.engine.cache.pages_free() == [m.engine.limits().num_pages]
    assert results[0] == results[1]
    # bfloat16 and eight bits together, one request alone, prompts that have nothing in common
    m = Model(ModelConfig(nr_ctx=512, max_tokens=4096, share_prefixes=True, cache_dtype="int8"))
    m.load(model_folders[name])
    m.init(top_k=40, top_p=0.95, temp=0.0, repeat_penalty=1.0, repeat_last_n=64, seed=1, end_token=2)
    for ps in (prompts, prompts[:1], [random_prompt(name, 70, 9), random_prompt(name, 80, 10)], [head, head, head]):
        out = m.generate(ps, max_new_tokens=6, stop_ids=[])
        assert [len(t) for t in out.tokens] == [6] * len(ps)
        m.engine.check_device_errors()
    assert out.tokens[0] == out.tokens[1] == out.tokens[2]


def test_adapters_and_shared_positions(model_folders):
    """Requests with different adapters share nothing: an adapter makes keys of its own."""
    name = "C"
    head = random_prompt(name, 150, 1)
    prompts = [head + random_prompt(name, 2 + i, 50 + i) for i in range(3)]
    tokens = []
    for share in (False, True):
        m = Model(ModelConfig(compt_type="float32", nr_ctx=512, max_tokens=4096, share_prefixes=share, max_adapters=2, adapter_rank=4))
        m.load(model_folders[name])
        m.init(top_k=40, top_p=0.95, temp=0.0, repeat_penalty=1.0, repeat_last_n=64, seed=1, end_token=2)
        g = torch.Generator().manual_seed(3)
        numbers = []
        for _ in range(2):
            names = {k: v for k, v in m.engine.adapted().items() if "k_proj" in k or "v_proj" in k}
            numbers.append(m.engine.add_adapter({k: (torch.randn((4, v[1]), generator=g) * v[1] ** -0.5, torch.randn((v[0], 4), generator=g) * 0.2) for k, v in names.items()}))
        tokens.append([m.generate(prompts, 6, stop_ids=[], adapters=a).tokens for a in ([numbers[0], numbers[1], -1], [numbers[1]] * 3)])
        m.engine.check_device_errors()
    assert tokens[0] == tokens[1]


def some_adapters(e, n):
    g = torch.Generator().manual_seed(5)
    shapes = {k: v for k, v in e.adapted().items() if "k_proj" in k or "q_proj" in k or "down_proj" in k}
    return [e.add_adapter({k: (torch.randn((4, v[1]), generator=g) * v[1] ** -0.5, torch.randn((v[0], 4), generator=g) * 0.2) for k, v in shapes.items()}) for _ in range(n)]


@pytest.mark.parametrize("cache", ["auto", "int8"])
@pytest.mark.parametrize("graphs", [True, False])
def test_adapters_beside_a_plan_of_common_positions(cache, graphs, model_folders):
    """Steps that bring both plans, eager and captured, with groups that change: as the steps that walk every sequence by itself."""
    name, got = "C", []
    prompt = random_prompt(name, 300, 1)
    for least in (0, 2 ** 62):
        e = engine(model_folders[name], cache=cache, cuda_graphs=graphs, max_batch=8, shared_prefix_bytes=least, max_adapters=2, adapter_rank=4)
        one, two = some_adapters(e, 2)
        a = e.new_sequence()
        e.step([StepItem(a, prompt, [], one)])
        slots = [a] + [e.fork_sequence(a, 256) for _ in range(4)]
        lone = e.new_sequence()
        e.step([StepItem(s, random_prompt(name, 3 + i, 10 + i), [], one) for i, s in enumerate(slots[1:])] + [StepItem(lone, prompt[:40], [], two)])
        out = []
        for j in range(6):
            order = slots + [lone] if j != 4 else [lone] + slots[::-1]
            logits = e.step([StepItem(s, random_prompt(name, 1, 100 + 10 * j + slots.index(s) if s != lone else 99), [0], two if s == lone else one) for s in order]).cpu().numpy()
            out += [logits[order.index(s)] for s in slots + [lone]]
        e.check_device_errors()
        got.append(np.stack(out))
    assert_close(got[0], got[1], "bfloat16")


def test_adapters_over_rows_of_eight_bits(model_folders):
    """In float32 a request's tokens do not depend on what else is in the step."""
    e = engine(model_folders["C"], "float32", max_batch=8, max_adapters=2, adapter_rank=4)
    one, two = some_adapters(e, 2)
    requests = [(random_prompt("C", 40 + 9 * i, i), a) for i, a in enumerate((one, two, -1))]

    def run(some):
        slots, out = [e.new_sequence() for _ in some], []
        out.append(e.step([StepItem(s, p, [len(p) - 1], a) for s, (p, a) in zip(slots, some)]).cpu())
        for j in range(4):
            out.append(e.step([StepItem(s, random_prompt("C", 1, 50 + j), [0], a) for s, (_, a) in zip(slots, some)]).cpu())
        for s in slots:
            e.end_sequence(s)
        return torch.stack(out, 1)

    together = run(requests)
    for i, r in enumerate(requests):
        assert_close(run([r])[0].numpy(), together[i].numpy(), "float32")
    assert (together[0] - together[2]).abs().max() > 0
    e.check_device_errors()


def test_the_cache_takes_half_the_room(model_folders):
    pages = [engine(model_folders["C"], cache=c, max_tokens=None, mem_fraction=0.02, max_batch=4).limits().num_pages for c in ("auto", "int8")]
    assert 1.85 <= pages[1] / pages[0] <= 2 * 128 / 132 + 0.01


def test_refusals(model_folders):
    with pytest.raises(EngineError, match="cache_dtype"):
        engine(model_folders["A"], cache="int4")
    with pytest.raises(EngineError, match="eight bits"):
        Engine.from_config(_windowless_none(), EngineOptions(cache_dtype="int8", max_tokens=256))
    e = engine(model_folders["D"])
    s = e.new_sequence()
    e.step([StepItem(s, random_prompt("D", 100, 1), [])])
    for length in (0, 1, 63, 65, 128, -64):
        with pytest.raises(CacheError):
            e.fork_sequence(s, length)
    with pytest.raises(CacheError):
        e.fork_sequence(s + 1, 64)
    assert e.sequence_length(e.fork_sequence(s, 64)) == 64


def _windowless_none():
    """A model none of whose layers keeps plain keys and values."""
    from plain_kudonex import random_config
    from inferllm_b200 import config_from_dict
    return config_from_dict(random_config(("mlstm", "attention")))


def test_command_line(model_folders):
    out = subprocess.run([f"{ROOT}/bin/llama", "-m", model_folders["C"], "-g", "GPU", "--prompt-ids", ",".join(map(str, range(1, 80))), "--prompt-ids",
                          ",".join(map(str, range(1, 70))), "-n", "4", "--temp", "0", "--cache-dtype", "int8", "--share-prefixes", "-c", "256", "--no-stop"],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    bad = subprocess.run([f"{ROOT}/bin/llama", "-m", model_folders["C"], "--prompt-ids", "1,2", "-n", "1", "--cache-dtype", "int3"], capture_output=True, text=True, timeout=300)
    assert bad.returncode != 0 and "cache_dtype" in bad.stderr


def test_a_step_of_more_sequences_than_a_plan_takes(model_folders):
    """It reads common positions for every sequence, and the pages that it brings are the sequences' own."""
    n = 65600
    e = engine(model_folders["C"], max_tokens=64 * (n + 70), max_batch=n + 2, max_seq_len=192, shared_prefix_bytes=0)
    prompt, last = random_prompt("C", 64, 1), random_prompt("C", 1, 2)
    a = e.new_sequence()
    e.step([StepItem(a, prompt, [])])
    slots = [e.fork_sequence(a, 64) for _ in range(n)]
    free = e.cache.pages_free()
    some = [0, 1, 32768, 65535, 65536, n - 1]
    got = e.step([StepItem(s, last, [0] if i in some else []) for i, s in enumerate(slots)]).cpu().numpy()
    e.check_device_errors()
    assert e.cache.pages_free() == [f - n for f in free]
    alone = e.step([StepItem(a, last, [0])]).cpu().numpy()
    for i in range(len(some)):
        assert_close(got[i:i + 1], alone, "bfloat16", f"sequence {some[i]}")
    e.cache.check()


@pytest.mark.parametrize("cache", ["auto", "int8"])
def test_steps_follow_the_rule_of_what_common_positions_save(cache, model_folders):
    """Behind 960 positions of two kv heads 300 sequences are on one side of the rule and 100 on the other, whatever the rows' type."""
    e = engine(model_folders["C"], cache=cache, cuda_graphs=False, max_tokens=64 * 330, max_batch=301)
    other = engine(model_folders["C"], cache=cache, cuda_graphs=False, max_tokens=64 * 330, max_batch=301, shared_prefix_bytes=2 ** 62)
    prompt, launches, got = random_prompt("C", 960, 1), {}, {}
    for which, x in (("rule", e), ("one by one", other)):
        a = x.new_sequence()
        x.step([StepItem(a, prompt, [])])
        slots = [x.fork_sequence(a, 960) for _ in range(300)]
        for n in (300, 100):
            before = ops.launch_count()
            got[which, n] = x.step([StepItem(s, [5], [0]) for s in slots[:n]]).cpu().numpy()
            launches[which, n] = ops.launch_count() - before
        x.check_device_errors()
    assert launches["rule", 300] > launches["one by one", 300] and launches["rule", 100] == launches["one by one", 100]
    for n in (300, 100):
        assert_close(got["rule", n], got["one by one", n], "bfloat16", f"{n} sequences")


def test_shared_positions_are_not_run_again(model_folders):
    """What the loop ran, by its own counts and the cache's: with and without sharing, with one adapter for all requests and with several, and through the command."""
    name = "C"
    head = random_prompt(name, 150, 1)
    prompts = [head + random_prompt(name, 2 + i, 50 + i) for i in range(5)]
    total = sum(map(len, prompts))
    for share in (False, True):
        m = Model(ModelConfig(compt_type="float32", nr_ctx=512, max_tokens=4096, share_prefixes=share, max_adapters=2, adapter_rank=4))
        m.load(model_folders[name])
        m.init(top_k=40, top_p=0.95, temp=0.0, repeat_penalty=1.0, repeat_last_n=64, seed=1, end_token=2)
        one, two = some_adapters(m.engine, 2)
        for adapters, shared in ((None, True), ([one] * 5, True), ([one, one, two, one, one], False), ([one, -1, -1, -1, -1], False)):
            used = []
            res = m.generate(prompts, 4, stop_ids=[], adapters=adapters, on_token=lambda r, t: used.append(m.engine.limits().num_pages - m.engine.cache.pages_free()[0]))
            n = 4 * 128 if share and shared else 0
            assert (res.prefill_tokens, res.shared_tokens) == (total - n, n)
            assert max(used) == 5 * 3 - n // 64
    for extra in ([], ["--share-prefixes"]):
        ids = [x for i in range(5) for x in ("--prompt-ids", ",".join(map(str, list(range(1, 80)) + [100 + i])))]
        out = subprocess.run([f"{ROOT}/bin/llama", "-m", model_folders[name], "-g", "GPU", *ids, "-n", "4", "--temp", "0", "-c", "256", "--no-stop", *extra],
                             capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr
        assert (f"prefill: {5 * 80 - 4 * 64} tokens" in out.stderr and "256 more held in common" in out.stderr) if extra else f"prefill: {5 * 80} tokens" in out.stderr


def test_the_engine_names_the_kernels_of_rows_in_eight_bits(model_folders):
    """What it says of itself: the kernels of the cache that it has, and a warning where these are the plain ones."""
    def says(name, *extra, **env):
        out = subprocess.run([f"{ROOT}/bin/llama", "-m", model_folders[name], "-g", "GPU", "--prompt-ids", "1,2,3", "-n", "1", "-c", "128", "--no-stop", *extra],
                             capture_output=True, text=True, timeout=300, env={**os.environ, **env})
        assert out.returncode == 0, out.stderr
        return out.stderr
    assert "rows of eight bits, prompts: tiles (tcgen05); single tokens: pages (TMA ring)" in says("C", "--cache-dtype", "int8", ILLM_LOG="info")
    assert "cache: 2 of 2 entries in eight bits" in says("C", "--cache-dtype", "int8", ILLM_LOG="info")
    assert "eight bits" not in says("C", ILLM_LOG="info") and "warning" not in says("C", "--cache-dtype", "int8")
    told = says("B", "--cache-dtype", "int8")
    assert "warning" in told and "rows of eight bits, prompts: plain" in told


@dataclass
class WideBeside(ArchConfig):
    """A layer with biases, whose entry stays in the activations' type, between two that can keep eight bits."""

    @classmethod
    def from_dict(cls, d):
        return cls()

    def to_dict(self):
        return {"architectures": ["WideBesideForCausalLM"]}

    def model_spec(self):
        norm = PartSpec("rmsnorm", {"size": HIDDEN, "eps": 1e-5})
        half = PartSpec("rope_half", {"head_dim": SIZE, "theta": BASE, "max_positions": 512})
        shape = {"hidden_size": HIDDEN, "n_heads": HEADS, "n_kv_heads": KV_HEADS, "head_dim": SIZE, "position": half}
        ffn = PartSpec("gated_mlp", {"hidden_size": HIDDEN, "intermediate_size": 128})
        layers = [LayerSpec("prenorm", PartSpec("attention", dict(shape, **more)), ffn, {"norm1": norm, "norm2": norm}, f"blocks.{i}.",
                            {"mixer": "mixer.", "ffn": "ffn.", "norm1": "ln1.", "norm2": "ln2."}) for i, more in enumerate(({}, {"qkv_bias": True}, {}))]
        return ModelSpec(HIDDEN, WORDS, layers, [ScheduleEntry(i, i) for i in range(3)], PartSpec("embedding", {"name": "emb.", "vocab_size": WORDS, "hidden_size": HIDDEN}),
                         PartSpec("rmsnorm", {"name": "ln_f.", "size": HIDDEN, "eps": 1e-5}),
                         PartSpec("lm_head", {"name": "head.", "tied": True, "vocab_size": WORDS, "hidden_size": HIDDEN}), 512, None, [])


def plain_beside(w, ids, rounds):
    pos, x = np.arange(len(ids)), plain.embed(ids, w["emb.weight"])
    for layer in range(3):
        p = f"blocks.{layer}."
        h = plain.rms_norm(x, w[p + "ln1.weight"], 1e-5)
        q, k, v = (plain.linear(h, w[p + f"mixer.{n}_proj.weight"]) + (w[p + f"mixer.{n}_proj.bias"] if layer == 1 else 0) for n in "qkv")
        q, k, v = (t.reshape(len(ids), -1, SIZE) for t in (q, k, v))
        angle = pos[:, None] * BASE ** (-np.arange(0, SIZE, 2) / SIZE)

        def turn(t):
            a, b, c, s = t[..., :SIZE // 2], t[..., SIZE // 2:], np.cos(angle)[:, None], np.sin(angle)[:, None]
            return np.concatenate([a * c - b * s, a * s + b * c], -1)
        q, k = turn(q), turn(k)
        if rounds and layer != 1:
            k, v = eight_bits(k), eight_bits(v)
        s = plain.scale_and_mask(plain.attention_scores(q, k, HEADS, KV_HEADS), SIZE ** -0.5)
        x = x + plain.linear(plain.weighted_values(plain.softmax_rows(s), v, HEADS, KV_HEADS), w[p + "mixer.o_proj.weight"])
        h = plain.rms_norm(x, w[p + "ln2.weight"], 1e-5)
        x = x + plain.swiglu_ffn(h, *(w[p + f"ffn.{n}_proj.weight"] for n in ("gate", "up", "down")))
    return plain.linear(plain.rms_norm(x, w["ln_f.weight"], 1e-5), w["emb.weight"])


@pytest.mark.parametrize("cache", ["auto", "int8"])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("n", [3, 60])
def test_common_positions_beside_a_layer_that_reads_them_one_by_one(cache, graphs, n, tmp_path):
    """Forks in a model whose layers differ: entries in eight bits, one that stays wide and whose layer takes no plan."""
    register_architecture("WideBesideForCausalLM", WideBeside)
    try:
        write_random_model(WideBeside(), str(tmp_path), seed=7, dtype=torch.bfloat16)
        _, w = plain.load_weights(str(tmp_path))
        e = engine(str(tmp_path), cache=cache, cuda_graphs=graphs, max_tokens=64 * (2 * n + 8), max_batch=n + 2, shared_prefix_bytes=0)
        groups = e.cache.stats()["paged"]
        assert sorted((bool(g["request"].get("int8")), len(g["entries"])) for g in groups) == ([(False, 1), (True, 2)] if cache == "int8" else [(False, 3)])
        R = np.random.default_rng(3)
        prompt = R.integers(0, WORDS, 150).tolist()
        a = e.new_sequence()
        e.step([StepItem(a, prompt, [])])
        slots, texts = [a] + [e.fork_sequence(a, 128) for _ in range(n - 1)], [list(prompt)] + [prompt[:128] for _ in range(n - 1)]
        more = [R.integers(0, WORDS, 1 + i % 9).tolist() for i in range(n - 1)]
        e.step([StepItem(s, t, []) for s, t in zip(slots[1:], more)])
        texts[1:] = [t + m for t, m in zip(texts[1:], more)]
        for j in range(4):
            tokens = [[int(t)] for t in R.integers(0, WORDS, n)]
            texts = [t + x for t, x in zip(texts, tokens)]
            got = e.step([StepItem(s, x, [0]) for s, x in zip(slots, tokens)]).cpu().numpy()
            for i in (0, 1, n - 1):
                assert_close(got[i:i + 1], plain_beside(w, texts[i], cache == "int8")[-1:], "bfloat16", f"token {j} of {i}")
        e.check_device_errors()
        assert (e.info()["graphs_captured"] > 0) == graphs
    finally:
        unregister_architecture("WideBesideForCausalLM")


def test_kinds_of_steps_that_came_once_do_not_push_captured_ones_out(model_folders):
    """Sequences that grow and batches that shrink make steps of many kinds; those that come again are replayed all the same."""
    e = engine(model_folders["C"], max_tokens=64 * 200, max_batch=80, shared_prefix_bytes=0)
    a = e.new_sequence()
    e.step([StepItem(a, random_prompt("C", 64, 1), [])])
    slots = [a] + [e.fork_sequence(a, 64) for _ in range(79)]
    for n in range(2, 80):                # 78 kinds, once each
        e.step([StepItem(s, [5], [0]) for s in slots[:n]])
    assert e.info()["graphs_captured"] == 0
    for _ in range(3):
        for n in (3, 40):
            got = e.step([StepItem(s, [5], [0]) for s in slots[-n:]])
    assert e.info()["graphs_captured"] >= 2 and torch.isfinite(got).all()
    e.check_device_errors()
