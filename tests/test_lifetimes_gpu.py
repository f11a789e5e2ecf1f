"""When engines and what belongs to them go (GPU): as soon as they are let go, never in the middle of a step that is being captured."""
import gc
import weakref
from dataclasses import dataclass

import pytest
import torch
from conftest import random_prompt

from inferllm_b200 import Engine, EngineOptions, Model, ModelConfig, StepItem, write_random_model
from inferllm_b200.config import ArchConfig, LayerSpec, ModelSpec, PartSpec, ScheduleEntry, register_architecture, unregister_architecture
from inferllm_b200.kernels import ops
from inferllm_b200.parts import PartSandbox, PositionEncoding, register_position, unregister_part

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, SIZE, WORDS = 64, 2, 32, 50


@pytest.fixture
def uncollected():
    """What is in no cycle goes without a collector."""
    gc.collect()
    gc.disable()
    yield
    gc.enable()


def test_an_engine_goes_when_it_is_let_go(uncollected, model_folders):
    e = Engine.from_folder(model_folders["A"], EngineOptions(max_tokens=256, max_batch=2))
    s = e.new_sequence()
    e.step([StepItem(s, random_prompt("A", 9, 1), [8])])
    assert e.cache is e.cache and e.cache.pages_free() == [256 // 64 - 1]
    cache, gone = e.cache, weakref.ref(e)
    del e
    assert gone() is not None and cache.pages_free() == [256 // 64 - 1]       # the cache's face holds its engine
    del cache
    assert gone() is None


def test_a_sandbox_goes_when_it_is_let_go(uncollected):
    box = PartSandbox({}, "float32")
    slots, gone = box.cache.slots_free, weakref.ref(box)
    assert slots
    del box
    assert gone() is None


@dataclass
class OnePart(ArchConfig):
    """A model whose layer has a position encoding of the test's."""

    @classmethod
    def from_dict(cls, d):
        return cls()

    def to_dict(self):
        return {"architectures": ["OnePartForCausalLM"]}

    def model_spec(self):
        norm = PartSpec("rmsnorm", {"size": HIDDEN, "eps": 1e-5})
        mixer = PartSpec("attention", {"hidden_size": HIDDEN, "n_heads": HEADS, "n_kv_heads": HEADS, "head_dim": SIZE, "position": PartSpec("lets_go_of_a_test", {})})
        ffn = PartSpec("gated_mlp", {"hidden_size": HIDDEN, "intermediate_size": 96})
        layers = [LayerSpec("prenorm", mixer, ffn, {"norm1": norm, "norm2": norm}, "blocks.0.", {"mixer": "mixer.", "ffn": "ffn.", "norm1": "ln1.", "norm2": "ln2."})]
        return ModelSpec(HIDDEN, WORDS, layers, [ScheduleEntry(0, 0)], PartSpec("embedding", {"name": "emb.", "vocab_size": WORDS, "hidden_size": HIDDEN}),
                         PartSpec("rmsnorm", {"name": "ln_f.", "size": HIDDEN, "eps": 1e-5}),
                         PartSpec("lm_head", {"name": "head.", "tied": True, "vocab_size": WORDS, "hidden_size": HIDDEN}), 256, None, [])


class LetsGo(PositionEncoding):
    """Lets go of other engines and models while its own engine's step is being captured."""
    others = []
    captures = 0

    def encode_and_store(self, qkv, geometry, ctx, kv):
        nh, nkv, d = geometry
        if torch.cuda.is_current_stream_capturing():
            LetsGo.captures += 1
            LetsGo.others.clear()
            gc.collect()
        ops.rope_kv_write(qkv, None, 0, ctx.token_pos, ctx.token_seq, kv.block_table, kv.k, kv.v, nh, nkv, d, kv.page_size, True, ctx.err)
        return qkv


@pytest.fixture
def one_part(tmp_path):
    register_architecture("OnePartForCausalLM", OnePart)
    register_position("lets_go_of_a_test")(LetsGo)
    write_random_model(OnePart(), str(tmp_path), seed=3, dtype=torch.bfloat16)
    yield str(tmp_path)
    unregister_architecture("OnePartForCausalLM")
    unregister_part("position", "lets_go_of_a_test")


def test_what_goes_while_a_step_is_captured_waits_for_its_end(one_part, model_folders):
    e = Engine.from_folder(one_part, EngineOptions(dtype="float32", max_tokens=256, max_batch=2, cuda_graphs=True))
    eager = Engine.from_folder(one_part, EngineOptions(dtype="float32", max_tokens=256, max_batch=2, cuda_graphs=False))
    other, m = Engine.from_folder(model_folders["A"], EngineOptions(max_tokens=256, max_batch=2)), Model(ModelConfig(nr_ctx=128, max_tokens=256))
    m.load(model_folders["A"])
    ring = [other, m, m.engine]
    ring.append(ring)
    gone = weakref.ref(other), weakref.ref(m)
    LetsGo.others, LetsGo.captures = [ring], 0
    del other, m, ring
    slots = e.new_sequence(), eager.new_sequence()
    for t in range(5):
        got, want = (x.step([StepItem(s, [t + 1], [0])]).cpu() for x, s in zip((e, eager), slots))
        assert torch.equal(got, want)
        assert (gone[0]() is None) == (LetsGo.captures > 0) == (gone[1]() is None)
    assert LetsGo.captures == 1 and e.info()["graphs_captured"] == 1
    e.check_device_errors()


def test_a_part_that_is_no_longer_registered_serves_the_engines_that_have_it(tmp_path):
    """Its callbacks stay until the last such engine has gone; the same kind may be registered anew beside it."""
    from inferllm_b200 import parts
    LetsGo.others = []
    made = []
    for _ in range(2):
        register_architecture("OnePartForCausalLM", OnePart)
        register_position("lets_go_of_a_test")(LetsGo)
        write_random_model(OnePart(), str(tmp_path), seed=3, dtype=torch.bfloat16)
        e = Engine.from_folder(str(tmp_path), EngineOptions(dtype="float32", max_tokens=256, max_batch=2))
        made.append((e, e.new_sequence()))
        unregister_architecture("OnePartForCausalLM")
        unregister_part("position", "lets_go_of_a_test")
        gc.collect()
    for t in range(4):
        a, b = (e.step([StepItem(s, [t + 1], [0])]).cpu() for e, s in made)
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert len(parts._UNREGISTERED) >= 2
    del e, made
    gc.collect()
    parts._retire("position", "none of this kind")
    assert not any(isinstance(x, LetsGo) for entry in parts._UNREGISTERED for x in entry[2].values())


def test_a_sampler_that_goes_while_its_engine_captures_waits_too(one_part):
    """Its buffers are freed behind what the engine's stream holds, which a stream that is being captured cannot be waited for."""
    from inferllm_b200.sampling import Sampler, SamplingParams
    e = Engine.from_folder(one_part, EngineOptions(dtype="float32", max_tokens=256, max_batch=2))
    sampler = Sampler(e, SamplingParams(temp=0.0, repeat_penalty=1.1, repeat_last_n=8))
    slot = e.new_sequence()
    logits = e.step([StepItem(slot, [1, 2, 3], [2])])
    token = sampler.choose(logits, [0], [0], [[1, 2, 3]])
    LetsGo.others, LetsGo.captures = [sampler], 0
    gone = weakref.ref(sampler)
    del sampler
    for t in range(4):
        got = e.step([StepItem(slot, [t + 1], [0])])
    assert LetsGo.captures == 1 and gone() is None and torch.isfinite(got).all() and 0 <= int(token[0]) < WORDS
    e.check_device_errors()


def test_the_cache_of_an_engine_that_has_gone_is_refused(model_folders):
    from inferllm_b200 import EngineError
    m = Model(ModelConfig(nr_ctx=128, max_tokens=256))
    m.load(model_folders["A"])
    old = m.engine
    assert old.cache.pages_free() == [4]
    m.load(model_folders["B"])
    with pytest.raises(EngineError, match="gone"):
        old.cache
    assert m.engine is not old and m.engine.cache.pages_free() == [4]
