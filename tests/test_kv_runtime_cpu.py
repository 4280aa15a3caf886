"""Refusals of the engine's cache and sampling settings without a GPU."""

import pytest
import torch
import torch.nn as nn


class _Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = nn.Linear(4, 4)
        self.register_buffer("at", torch.zeros(1))

    def generate(self, input_ids=None, max_new_tokens=1, **kw):
        self.seen = kw
        return torch.cat([input_ids, torch.zeros(input_ids.shape[0], max_new_tokens, dtype=input_ids.dtype)], dim=1)


@pytest.mark.filterwarnings("ignore:.*0 hooked layers")
def test_engine_refuses_what_it_cannot_do():
    from csaq.inference import CSAQInferenceEngine
    with pytest.raises(ValueError, match="kv_bits"):
        CSAQInferenceEngine(_Model(), {}, verbose=False, kv_bits=3)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    eng = CSAQInferenceEngine(_Model(), {}, verbose=False, kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits"):  # no decode runtime for this model
        eng.generate(ids, max_new_tokens=2, temperature=0.0)
    eng = CSAQInferenceEngine(_Model(), {}, verbose=False)
    with pytest.raises(ValueError, match="runtime"):
        eng.generate(ids, max_new_tokens=2, random=torch.zeros(2, 2))
    with pytest.raises(ValueError, match="speculative"):
        eng.generate(ids, max_new_tokens=2, speculative=True, random=torch.zeros(2, 2))


@pytest.mark.filterwarnings("ignore:.*0 hooked layers")
def test_settings_still_reach_the_model_without_random_numbers():
    from csaq.inference import CSAQInferenceEngine
    model = _Model()
    out, rep = CSAQInferenceEngine(model, {}, verbose=False).generate(
        torch.zeros(1, 3, dtype=torch.int64), max_new_tokens=2, temperature=0.7, top_k=5, min_p=0.1)
    assert out.shape == (1, 5) and rep.mode == "standard"
    assert model.seen["top_k"] == 5 and model.seen["min_p"] == 0.1 and model.seen["temperature"] == 0.7
