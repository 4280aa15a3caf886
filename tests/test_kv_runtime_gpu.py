"""The decode runtime with a quantised KV cache, and decoding from given random numbers.

* Prefill in one chunk (the cache read back for torch's attention) and in chunks
  that go through attention over the codes agree, at the bound that the runtime's
  logits are held to against HF (two bf16 evaluations of one computation).
* What a layer's cache holds after a prefill is the definition's, from the
  projections of the model's own first layer.
* Greedy self-speculative decoding equals greedy decoding with the verify weights
  token for token: a token's attention does not depend on the step's tokens.
* Every sampled token is the one that the 64-bit reference draws from the step's
  own logits.
"""

import numpy as np
import pytest
import torch

import _kv_ref
import _sample_ref
from test_runtime_gpu import _prompt, _quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def models():
    return {"tiny-llama": _quantized("tiny-llama"), "tiny-qwen2-d64": _quantized("tiny-qwen2-d64", seed=6)}


def _engine(models, name, **kw):
    from csaq.inference import CSAQInferenceEngine
    model, cmap, _ = models[name]
    return CSAQInferenceEngine(model, cmap, verbose=False, **kw)


@pytest.mark.parametrize("name,bits", [("tiny-llama", 8), ("tiny-llama", 4), ("tiny-qwen2-d64", 8)])
def test_prefill_chunks_agree(models, name, bits):
    eng = _engine(models, name, kv_bits=bits)
    rt = eng.runtime(2, 256, 4)
    prompt = _prompt(2, 70, eng.model.config.vocab_size, seed=3).to(DEV)
    rt.reset(prompt, max_new=4)  # one chunk
    want, caches = rt.prefill_logits.float(), [t.clone() for t in rt.kvq[0].buffers()]
    for chunk in (32, 16):  # 32 + 32 + 6, and 16s: attention over the codes
        rt.prefill_chunk = chunk
        rt.reset(prompt, max_new=4)
        got = rt.prefill_logits.float()
        assert (got - want).abs().max() / want.abs().max() < 3e-2
        assert (torch.nn.functional.cosine_similarity(got, want) > 0.999).all()
        # the first layer's projections do not depend on attention: their codes neither
        # (the GEMV serves both chunk lengths)
        if chunk == 16:
            assert all(torch.equal(a, b) for a, b in zip(rt.kvq[0].buffers(), small))
        small = [t.clone() for t in rt.kvq[0].buffers()]
    assert caches[0].shape[2] == rt.kvq[0].max_len
    rt.prefill_chunk = 512


def test_the_cache_holds_the_definition(models):
    """Layer 0: keys and values of the runtime's own fused projection, rotated and stored."""
    eng = _engine(models, "tiny-llama", kv_bits=8)
    rt = eng.runtime(2, 128, 4)
    P = 20
    rt.reset(_prompt(2, P, eng.model.config.vocab_size, seed=5).to(DEV), max_new=2)
    c, D, Hkv, nq = rt.kvq[0], rt.D, rt.Hkv_l, rt.Hq_l * rt.D
    # run layer 0's projection again on the same input
    sh = rt.shapes[P]
    ids = _prompt(2, P, eng.model.config.vocab_size, seed=5).to(DEV).view(-1)
    from csaq._lib import check, lib
    st = torch.cuda.current_stream().cuda_stream
    torch.index_select(rt.embed, 0, ids, out=sh.x)
    check(lib().csaq_rmsnorm(sh.x.data_ptr(), rt.H, rt.layers[0].input_layernorm.weight.data_ptr(), sh.xn.data_ptr(), rt.H,
                             sh.M, rt.H, rt.eps, rt.dt, st), "rmsnorm")
    rt._gemv(sh.descs[(0, "qkv", True)], rt.H, sh.xn, sh.M, st)
    kv = sh.qkv[:, nq:].float().cpu().numpy().reshape(2, P, 2, Hkv, D)
    cos, sin = rt.cos[:P].cpu().numpy()[None, :, None], rt.sin[:P].cpu().numpy()[None, :, None]
    for i, x in enumerate((_kv_ref.rotate(kv[:, :, 0], cos, sin), kv[:, :, 1])):
        codes, words = _kv_ref.quantise(x.transpose(0, 2, 1, 3), 8, c.group_size)
        assert np.array_equal(c.buffers()[2 * i][:, :, :P].cpu().numpy(), codes.astype(np.uint8))
        assert np.array_equal(c.buffers()[2 * i + 1][:, :, :P].cpu().numpy(), words.view(np.int32))


@pytest.mark.parametrize("name,B,K,bits", [("tiny-llama", 1, 4, 8), ("tiny-llama", 3, 4, 4), ("tiny-llama", 16, 4, 8),
                                           ("tiny-qwen2-d64", 2, 6, 8)])
def test_speculative_equals_greedy(models, name, B, K, bits):
    eng = _engine(models, name, kv_bits=bits)
    prompt = _prompt(B, 33, eng.model.config.vocab_size, seed=7 + B)
    out, rep = eng.generate(prompt, speculative=True, lookahead=K, temperature=0.0, max_new_tokens=40)
    assert out.shape == (B, 73) and rep.verify_calls > 0
    rt = eng.runtime(B, 33 + 40 + 2 * K + 2, K)
    assert rt.kv_bits == bits and rt.k_cache is None
    rt.reset(prompt.to(DEV), 40, verify=True)
    rt.generate_greedy(40, verify=True)
    assert torch.equal(out[:, 33:].cpu(), rt.outputs()[:, :40].cpu())


@pytest.mark.parametrize("name,bits", [("tiny-llama", 8), ("tiny-llama", 4), ("tiny-qwen2-d64", 8)])
def test_contexts_of_several_chunks(models, name, bits):
    """400 positions, which attention takes in four chunks of keys: prefill in pieces agrees
    with prefill in one, the decode steps write nothing but their outputs, and speculation
    equals greedy decoding."""
    eng = _engine(models, name, kv_bits=bits)
    P, n, K = 400, 40, 4
    rt = eng.runtime(2, P + n + 2 * K + 2, K)
    prompt = _prompt(2, P, eng.model.config.vocab_size, seed=9).to(DEV)
    rt.reset(prompt, max_new=n)
    want = rt.prefill_logits.float()
    rt.prefill_chunk = 16
    rt.reset(prompt, max_new=n)
    rt.prefill_chunk = 512
    got = rt.prefill_logits.float()
    assert (got - want).abs().max() / want.abs().max() < 3e-2
    assert (torch.nn.functional.cosine_similarity(got, want) > 0.999).all()
    rt.reset(prompt, n, verify=True)
    held = [[t[:, :, :P].clone() for t in c.buffers()] for c in rt.kvq]
    weights = {k: v.clone() for k, v in eng.model.state_dict().items()}
    rt.generate_greedy(n, verify=True)
    assert all(torch.equal(t[:, :, :P], o) for c, old in zip(rt.kvq, held) for t, o in zip(c.buffers(), old))
    assert all(torch.equal(v, weights[k]) for k, v in eng.model.state_dict().items())
    greedy = rt.outputs()[:, :n].cpu()
    out, _ = eng.generate(prompt.cpu(), speculative=True, lookahead=K, temperature=0.0, max_new_tokens=n)
    assert torch.equal(out[:, P:].cpu(), greedy)


def test_speculative_sampling_runs(models):
    eng = _engine(models, "tiny-llama", kv_bits=8)
    prompt = _prompt(2, 12, eng.model.config.vocab_size, seed=1)
    a, _ = eng.generate(prompt, speculative=True, temperature=0.9, top_p=0.9, max_new_tokens=12, seed=3)
    b, _ = eng.generate(prompt, speculative=True, temperature=0.9, top_p=0.9, max_new_tokens=12, seed=3)
    assert a.shape == (2, 24) and torch.equal(a, b)


@pytest.mark.parametrize("bits", [None, 8])
def test_tokens_from_given_numbers(models, bits):
    eng = _engine(models, "tiny-llama", kv_bits=bits)
    V, B, P, N = eng.model.config.vocab_size, 3, 21, 14
    prompt = _prompt(B, P, V, seed=2)
    u = torch.rand(B, N, generator=torch.Generator().manual_seed(4))
    kw = dict(temperature=torch.tensor([0.8, 0.0, 1.2]), top_k=torch.tensor([50, 0, 0], dtype=torch.int32),
              top_p=torch.tensor([0.95, 1.0, 0.8]), min_p=torch.tensor([0.0, 0.0, 0.05]))
    out, rep = eng.generate(prompt, max_new_tokens=N, random=u, **kw)
    assert out.shape == (B, P + N) and torch.equal(out[:, :P], prompt) and rep.mode == "standard"
    assert rep.tokens_generated == B * N
    toks = out[:, P:]
    # teacher-forced: the same steps, each token drawn by the reference from the step's logits
    rt = eng.runtime(B, P + N + 4, 1)
    rt.reset(prompt.to(DEV), N, verify=False)
    logits = rt.prefill_logits
    for i in range(N):
        x = logits.double().cpu().numpy()
        for b in range(B):
            one = {k: v[b].item() for k, v in kw.items()}
            assert int(toks[b, i]) == _sample_ref.sample(x[b], float(u[b, i]), **one)[0], (b, i)
        rt.next_tok.copy_(toks[:, i])
        rt.step(1, rt.next_tok, rt.pos0, verify=False)
        logits = rt.logits_view(1, B).clone()
        rt.pos0.add_(1)
    # the same numbers again, and one sequence with other settings: only that one changes
    again, _ = eng.generate(prompt, max_new_tokens=N, random=u, **kw)
    assert torch.equal(again, out)
    kw["temperature"] = torch.tensor([0.8, 0.0, 30.0])
    other, _ = eng.generate(prompt, max_new_tokens=N, random=u, **kw)
    assert torch.equal(other[:2], out[:2]) and not torch.equal(other[2], out[2])


def test_one_number_draws_the_prefill_token(models):
    eng = _engine(models, "tiny-qwen2-d64", kv_bits=4)
    prompt = _prompt(1, 9, eng.model.config.vocab_size, seed=8)
    out, _ = eng.generate(prompt, max_new_tokens=1, temperature=0.7, top_k=5, random=torch.full((1, 1), 0.99))
    rt = eng.runtime(1, 9 + 1 + 4, 1)
    rt.reset(prompt.to(DEV), 1, verify=False)
    assert int(out[0, 9]) == _sample_ref.sample(rt.prefill_logits[0].double().cpu().numpy(), float(np.float32(0.99)),
                                                temperature=0.7, top_k=5)[0]


def test_steps_with_nothing_to_draw(models):
    """Logits of NaN: token 0, a row of the embedding, in the prefill's draw and the steps'."""
    eng = _engine(models, "tiny-llama", kv_bits=8)
    prompt, u = _prompt(2, 9, eng.model.config.vocab_size, seed=8), torch.full((2, 5), 0.5)
    want, _ = eng.generate(prompt, max_new_tokens=5, random=u)
    norm = eng.model.model.norm.weight.data
    kept = norm.clone()
    norm.fill_(float("nan"))
    try:
        out, _ = eng.generate(prompt, max_new_tokens=5, random=u)
    finally:
        norm.copy_(kept)
    assert (out[:, 9:] == 0).all() and torch.equal(out[:, :9], prompt)
    assert torch.equal(eng.generate(prompt, max_new_tokens=5, random=u)[0], want)


def test_tokens_are_drawn_once_after_a_reset(models):
    eng = _engine(models, "tiny-llama", kv_bits=8)
    rt = eng.runtime(1, 64, 1)
    rt.reset(_prompt(1, 6, eng.model.config.vocab_size, seed=1).to(DEV), 8)
    assert rt.generate_sampled(torch.full((1, 3), 0.5)) == 2
    with pytest.raises(RuntimeError, match="reset"):
        rt.generate_sampled(torch.full((1, 3), 0.5))


def test_kernel_counts_follow_the_cache(models):
    a, b = _engine(models, "tiny-llama"), _engine(models, "tiny-llama", kv_bits=8)
    ra, rb = a.runtime(1, 256, 4), b.runtime(1, 256, 4)
    assert rb.kernels_per_step(1) == ra.kernels_per_step(1) + ra.n_layers
    assert rb.prefill_kernels(100) == ra.prefill_kernels(100) + ra.n_layers


def test_refusals(models):
    from csaq.runtime import DecodeRuntime
    model = models["tiny-llama"][0]
    for kw in (dict(kv_bits=2), dict(kv_bits=16), dict(kv_group=64), dict(kv_bits=8, kv_group=32)):
        with pytest.raises(ValueError):
            DecodeRuntime(model, 1, 64, **kw)
    eng = _engine(models, "tiny-llama", kv_bits=8)
    prompt = _prompt(2, 6, model.config.vocab_size, seed=1)
    u = torch.zeros(2, 4)
    for kw, what in ((dict(random=u, speculative=True), "speculative"), (dict(random=u[:, :3]), "random"),
                     (dict(random=u, repetition_penalty=1.1), "repetition_penalty"), (dict(temperature=0.8), "kv_bits"),
                     (dict(random=u, top_p=0.0), "top_p"), (dict(random=u, top_k=torch.ones(3)), "top_k")):
        with pytest.raises(ValueError, match=what):
            eng.generate(prompt, max_new_tokens=4, **kw)
    rt = eng.runtime(2, 64, 1)
    rt.reset(prompt.to(DEV), 3)
    with pytest.raises(ValueError, match="random"):
        rt.generate_sampled(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="random"):
        rt.generate_sampled(torch.zeros(3, 2))
