"""What the decode runtime and the engine hold for a quantised cache."""

import pytest
import torch

from test_runtime_gpu import _prompt, _quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def model():
    return _quantized("tiny-llama")


def _engine(model, **kw):
    from csaq.inference import CSAQInferenceEngine
    return CSAQInferenceEngine(model[0], model[1], verbose=False, **kw)


def test_a_prompt_in_chunks_is_read_back_into_one_buffer(model):
    eng = _engine(model, kv_bits=8)
    rt = eng.runtime(2, 400, 4)
    rt.prefill_chunk = 64
    held = []
    inner = rt._sdpa
    rt._sdpa = lambda *a, **kw: (held.append((rt.kv_read.data_ptr(), rt.kv_read.numel())), inner(*a, **kw))[1]
    rt.reset(_prompt(2, 300, eng.model.config.vocab_size, seed=3).to(DEV), max_new=4)
    # 64 positions four times and 44
    assert len(held) == 5 * rt.n_layers and len(set(held)) == 1
    assert held[0][1] == 2 * 2 * rt.Hkv_l * 300 * rt.D  # keys and values of the prompt, no more
    first = rt.prefill_logits.clone()
    rt.reset(_prompt(2, 90, eng.model.config.vocab_size, seed=4).to(DEV), max_new=4)
    rt.reset(_prompt(2, 300, eng.model.config.vocab_size, seed=3).to(DEV), max_new=4)
    assert len(set(held)) == 1  # shorter prompts and repeats use it again
    assert torch.equal(rt.prefill_logits, first)
    rt._sdpa = inner


def test_steps_without_a_reset_get_a_buffer_too(model):
    """A caller of step() with its own positions: the buffer grows, at most twofold at a time and
    never beyond the cache."""
    eng = _engine(model, kv_bits=8)
    rt = eng.runtime(1, 256, 4)
    ids = _prompt(1, 256, eng.model.config.vocab_size, seed=5).to(DEV).view(-1)
    sizes = []
    for s0 in range(0, 256, 32):
        rt.pos0.fill_(s0)
        rt.step(32, ids[s0:s0 + 32].contiguous(), rt.pos0, verify=True, last_only=True, pos_host=s0)
        sizes.append(rt.kv_read.numel())
    assert len(set(sizes)) <= 5 and max(sizes) <= 2 * rt.Hkv_l * rt.Lmax * rt.D


def test_kv_bits_set_later_make_another_runtime(model):
    eng = _engine(model)
    prompt = _prompt(1, 12, eng.model.config.vocab_size, seed=1)
    eng.generate(prompt, temperature=0.0, max_new_tokens=4)
    assert eng._runtime.kv_bits is None
    eng.kv_bits = 8
    want, _ = eng.generate(prompt, temperature=0.0, max_new_tokens=4)
    assert eng._runtime.kv_bits == 8
    rt = eng._runtime
    u = torch.rand(1, 4, generator=torch.Generator().manual_seed(2))
    eng.generate(prompt, random=u, max_new_tokens=4)  # shares the runtime of one batch and cache
    assert eng._runtime is rt
    eng.kv_bits = None
    eng.generate(prompt, random=u, max_new_tokens=4)
    assert eng._runtime.kv_bits is None
    eng.kv_bits = 5
    with pytest.raises(ValueError, match="kv_bits"):
        eng.generate(prompt, temperature=0.0, max_new_tokens=4)
