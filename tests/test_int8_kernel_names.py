"""Which kernels a layer over rows of eight bits is said to get (no GPU)."""
import ctypes

import pytest

from inferllm_b200 import binding as _b

FLOAT32, BFLOAT16 = 0, 1


@pytest.mark.parametrize("dtype, heads, kv_heads, size, page, prompts, tokens", [
    (BFLOAT16, 32, 8, 128, 64, "tiles", "pages"), (BFLOAT16, 14, 2, 64, 128, "tiles", "pages"), (BFLOAT16, 32, 1, 128, 64, "tiles", "plain"),
    (BFLOAT16, 32, 8, 96, 64, "plain", "plain"), (BFLOAT16, 32, 8, 128, 16, "plain", "plain"), (FLOAT32, 32, 8, 128, 64, "plain", "plain")])
def test_names(dtype, heads, kv_heads, size, page, prompts, tokens):
    out = ctypes.c_void_p()
    _b.check(_b.lib().illm_policy_attention_kernels_int8(dtype, heads, kv_heads, size, page, ctypes.byref(out)))
    said = _b.take_string(out)
    assert said.startswith(f"rows of eight bits, prompts: {prompts} (") and f"; single tokens: {tokens} (" in said
