"""Timed cases of the quantised KV cache, the attention that reads it, and filtered sampling.

Each case is run either in its plain form (elementary torch operations) or,
with ``own`` set, through the package's public calls:

* ``write``: rotary embedding of a step's queries and keys, the keys and values
  quantised into the cache, and the written positions read back as the values
  they stand for (``QuantizedKVCache.write`` and ``.read``);
* ``read``: positions 0..n of a cache read back in the model's dtype, what a
  prefill over an existing cache does before its attention
  (``QuantizedKVCache.read``);
* ``attend``: causal grouped-query attention of a step's tokens against the
  quantised cache (``QuantizedKVCache.attend``);
* ``sample``: one token per logit row from a given random number under
  temperature, top-k, top-p and min-p (``sample_tokens``).

The cache's storage, which both forms read and write: per (token, head, group
of ``group`` head elements) one 32-bit word, the upper half the bf16 scale s,
the lower half 0x6400 + zero point z; codes c of 8 or 4 bits (4-bit: even
element in the low nibble); the value is s * (c - z).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    llama = {"Hq": 32, "Hkv": 8, "D": 128}     # the benchmark's 8B decoder
    qwen = {"Hq": 16, "Hkv": 16, "D": 64}      # its 0.5B decoder: one query head per KV head
    return [
        # one decode step of 16 sequences: latency of the smallest write
        {"name": "write_decode_b16", "op": "write", "B": 16, "S": 1, **llama, "bits": 8, "group": 128, "dtype": "bf16",
         "start": 700},
        # a batch of prompts, 4-bit in groups of 64
        {"name": "write_prefill_b16_2048_4bit", "op": "write", "B": 16, "S": 2048, **llama, "bits": 4, "group": 64,
         "dtype": "fp16", "start": 0},
        # the cache of a prompt in progress, read back for the next prefill chunk
        {"name": "read_b1_1999", "op": "read", "B": 1, "n": 1999, **llama, "bits": 8, "group": 128, "dtype": "bf16"},
        # long contexts of a batch, 4-bit
        {"name": "read_b8_32768_4bit", "op": "read", "B": 8, "n": 32768, **llama, "bits": 4, "group": 64,
         "dtype": "fp16"},
        # the benchmark's decode step: batch 1, 512-token prompt
        {"name": "attend_b1_517", "op": "attend", "B": 1, "S": 1, **llama, "bits": 8, "group": 128, "dtype": "bf16",
         "longest": 517, "ragged": False},
        # a speculative verify pass: 4 drafts and one more token for each of 4 sequences
        {"name": "attend_verify_b4_s5", "op": "attend", "B": 4, "S": 5, **llama, "bits": 8, "group": 64,
         "dtype": "bf16", "longest": 4101, "ragged": True},
        # a serving batch of unequal lengths
        {"name": "attend_b32_ragged_8192", "op": "attend", "B": 32, "S": 1, **llama, "bits": 8, "group": 128,
         "dtype": "bf16", "longest": 8192, "ragged": True},
        # 64-wide heads without sharing, fp16, 4-bit
        {"name": "attend_mha_d64_b16_4bit", "op": "attend", "B": 16, "S": 1, **qwen, "bits": 4, "group": 64,
         "dtype": "fp16", "longest": 6001, "ragged": True},
        # long contexts, where the cache's bytes are everything
        {"name": "attend_b8_65536_4bit", "op": "attend", "B": 8, "S": 1, **llama, "bits": 4, "group": 64,
         "dtype": "bf16", "longest": 65536, "ragged": False},
        # one user's next token, all filters on
        {"name": "sample_b1_topk_topp", "op": "sample", "rows": 1, "V": 128256, "dtype": "bf16", "top_k": 50,
         "top_p": 0.95, "min_p": 0.02, "temperature": 0.8, "mixed": False},
        # a serving batch, every row with its own settings
        {"name": "sample_b64_mixed", "op": "sample", "rows": 64, "V": 151936, "dtype": "bf16", "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "temperature": 1.0, "mixed": True},
        # many rows of an odd vocabulary in fp32, nucleus only
        {"name": "sample_b256_fp32_topp", "op": "sample", "rows": 256, "V": 50257, "dtype": "fp32", "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "temperature": 0.7, "mixed": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "sample"])
    if op == "sample":
        V = _log_int(rng, 1000, 160000)
        rows = _log_int(rng, 1, max(1, min(300, 10_000_000 // V)))
        return {"op": op, "rows": rows, "V": V, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "top_k": rng.choice([0, 0, _log_int(rng, 1, 2000)]), "top_p": rng.choice([1.0, rng.uniform(0.3, 0.99)]),
                "min_p": rng.choice([0.0, rng.uniform(0.001, 0.2)]), "temperature": rng.uniform(0.3, 1.5),
                "mixed": rng.random() < 0.3}
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    G = rng.choice([1, 2, 4, 7, 8])
    case = {"op": op, "Hq": Hkv * G, "Hkv": Hkv, "D": D, "bits": rng.choice([8, 4]),
            "group": rng.choice([64, D]), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "write":
        case["B"] = _log_int(rng, 1, 32)
        most = max(1, min(2048, 100_000_000 // (case["B"] * Hkv * G * D)))
        case["S"] = _log_int(rng, 1, most)
        case["start"] = rng.choice([0, _log_int(rng, 1, 4000)])
        return case
    case["B"] = _log_int(rng, 1, 48)
    most = max(64, min(60000, 200_000_000 // (case["B"] * Hkv * D)))
    if op == "read":
        case["n"] = _log_int(rng, 1, most)
        return case
    case["S"] = rng.choice([1, 1, 2, 5, 9])
    case["longest"] = _log_int(rng, case["S"], most)
    case["ragged"] = rng.random() < 0.6
    return case


# ── inputs ───────────────────────────────────────────────────────────────────

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rope_tables(n, D):
    inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
    f = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    f = torch.cat([f, f], dim=-1)
    return f.cos().float().contiguous(), f.sin().float().contiguous()


def _keys(g, *shape):
    """Keys as attention meets them: a few channels far larger than the others."""
    D = shape[-1]
    gain = torch.ones(D, device=DEV)
    gain[torch.randint(0, D, (max(1, D // 32),), generator=g, device=DEV)] = 6.0
    return _normal(g, *shape) * gain


def _capacity(n):
    return (n + 15) // 16 * 16


def prepare(case, seed):
    g = _generator(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    state = {"case": dict(case), "dtype": dt}
    if op == "sample":
        rows, V = case["rows"], case["V"]
        # a language model's logits: a broad bulk, a few likely tokens, some banned ones
        x = 2.5 * _normal(g, rows, V)
        hot = torch.randint(0, V, (rows, 24), generator=g, device=DEV)
        x.scatter_add_(1, hot, 6.0 + 3.0 * _normal(g, rows, 24))
        x.scatter_(1, torch.randint(0, V, (rows, 5), generator=g, device=DEV), float("-inf"))
        state["logits"] = x.to(dt)
        state["random"] = torch.rand(rows, generator=g, device=DEV)
        if case["mixed"]:  # a device tensor of each setting, as a server keeps them
            pick = torch.randint(0, 4, (4, rows), generator=g, device=DEV)
            of = lambda i, values, t: torch.tensor(values, dtype=t, device=DEV)[pick[i]]  # noqa: E731
            state["temperature"] = of(0, [0.6, 0.8, 1.0, 1.3], torch.float32)
            state["top_k"] = of(1, [0, 0, 40, 400], torch.int32)
            state["top_p"] = of(2, [1.0, 0.95, 0.9, 0.5], torch.float32)
            state["min_p"] = of(3, [0.0, 0.0, 0.05, 0.1], torch.float32)
        else:
            state.update({k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")})
        return state
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    bits, group = case["bits"], case["group"]
    if op == "write":
        S, start = case["S"], case["start"]
        L = _capacity(start + S)
        qkv = torch.cat([_normal(g, B * S, Hq * D), _keys(g, B * S, Hkv, D).view(B * S, Hkv * D),
                         _normal(g, B * S, Hkv * D)], dim=1).to(dt)  # one fused projection's output
        nq, nk = Hq * D, Hkv * D
        state["q"], state["k"], state["v"] = qkv[:, :nq], qkv[:, nq:nq + nk], qkv[:, nq + nk:]
        state["cos"], state["sin"] = _rope_tables(L, D)
        state["pos0"] = torch.full((B,), start, dtype=torch.int32, device=DEV)
        z = lambda *s, t: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
        for name in "kv":
            state[name + "_codes"] = z(B, Hkv, L, D * bits // 8, t=torch.uint8)
            state[name + "_params"] = z(B, Hkv, L, D // group, t=torch.int32)
        return state
    n = case["n"] if op == "read" else case["longest"]
    L = _capacity(n)
    for name, x in (("k", _keys(g, B, Hkv, L, D)), ("v", _normal(g, B, Hkv, L, D))):
        codes, scale, zero = _codes_of(x, bits, group)
        state[name + "_codes"] = _packed(codes, bits).contiguous()
        state[name + "_params"] = _words(scale, zero).contiguous()
        del x, codes, scale, zero
    if op == "attend":
        S = case["S"]
        state["q"] = _normal(g, B * S, Hq * D).to(dt)
        if case["ragged"]:
            low = max(0, (n - S) // 16)
            pos0 = torch.randint(low, n - S + 1, (B,), generator=g, device=DEV)
            pos0[torch.randint(0, B, (1,), generator=g, device=DEV)] = n - S
        else:
            pos0 = torch.full((B,), n - S, device=DEV)
        state["pos0"] = pos0.to(torch.int32)
    return state


# ── plain forms ──────────────────────────────────────────────────────────────

def _codes_of(x, bits, group):
    """(codes, scale, zero) of fp32 x (..., D): every operation is one fp32 rounding."""
    levels = float(2 ** bits - 1)
    xg = x.unflatten(-1, (-1, group))
    low = xg.amin(-1, keepdim=True).clamp(max=0.0)
    span = xg.amax(-1, keepdim=True).clamp(min=0.0) - low
    word = (span / torch.full_like(span, levels)).view(torch.int32)  # quotients by tensors: correctly rounded
    word = (word + 0xFFFF) & -0x10000                                # the bf16 scale, rounded up
    scale = torch.where(span > 0, word.clamp(min=0x00800000), 0).view(torch.float32)
    step = torch.where(scale > 0, scale, 1.0)
    zero = (-low / step).round().clamp(0.0, levels)
    codes = ((xg / step).round() + zero).clamp(0.0, levels)
    return codes.flatten(-2), scale.squeeze(-1), zero.squeeze(-1)


def _packed(codes, bits):
    c = codes.to(torch.uint8)
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def _words(scale, zero):
    return scale.view(torch.int32) | (0x6400 + zero.to(torch.int32))


def _values(codes, words, bits, group):
    """The fp32 values that packed codes and their words stand for."""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    scale = (words & -0x10000).view(torch.float32).unsqueeze(-1)
    zero = ((words & 0xFFFF) - 0x6400).unsqueeze(-1).float()
    return ((codes.unflatten(-1, (-1, group)).float() - zero) * scale).flatten(-2)


def _rotated(x, cos, sin):
    """rotate_half of x (..., D): products and their sum each rounded to fp32."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    ca, cb, sa, sb = cos[..., :half], cos[..., half:], sin[..., :half], sin[..., half:]
    return torch.cat([a * ca - b * sa, b * cb + a * sb], dim=-1)


def _plain_write(state):
    c = state["case"]
    B, S, Hq, Hkv, D, bits, group = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "bits", "group"))
    dt = state["dtype"]
    pos = state["pos0"].long()[:, None] + torch.arange(S, device=DEV)
    cos, sin = state["cos"][pos][:, :, None], state["sin"][pos][:, :, None]      # (B, S, 1, D)
    heads = lambda x, h: x.float().view(B, S, h, D)                              # noqa: E731
    q = _rotated(heads(state["q"], Hq), cos, sin).to(dt).view(B * S, Hq * D)
    k = _rotated(heads(state["k"], Hkv), cos, sin).transpose(1, 2).contiguous()  # (B, Hkv, S, D)
    v = heads(state["v"], Hkv).transpose(1, 2).contiguous()
    (kc, ks, kz), (vc, vs, vz) = _codes_of(k, bits, group), _codes_of(v, bits, group)
    back = lambda codes, s, z: _values(_packed(codes, bits), _words(s, z), bits, group).to(dt)  # noqa: E731
    return {"q": q, "k": back(kc, ks, kz), "v": back(vc, vs, vz)}


def _plain_read(state):
    c = state["case"]
    part = lambda name: _values(state[name + "_codes"][:, :, :c["n"]], state[name + "_params"][:, :, :c["n"]],  # noqa: E731
                                c["bits"], c["group"]).to(state["dtype"])
    return {"k": part("k"), "v": part("v")}


def _plain_attend(state):
    c = state["case"]
    B, S, Hq, Hkv, D = (c[k] for k in ("B", "S", "Hq", "Hkv", "D"))
    q = state["q"].float().view(B, S, Hkv, Hq // Hkv, D)
    k = _values(state["k_codes"], state["k_params"], c["bits"], c["group"])
    L = k.shape[2]
    last = state["pos0"].long()[:, None] + torch.arange(S, device=DEV)           # (B, S): the last visible key
    seen = torch.arange(L, device=DEV) <= last[:, :, None]                       # (B, S, L)
    w = torch.einsum("bshgd,bhld->bhsgl", q, k) * (1.0 / math.sqrt(D))
    del k
    w = w.masked_fill(~seen[:, None, :, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    v = _values(state["v_codes"], state["v_params"], c["bits"], c["group"])
    out = torch.einsum("bhsgl,bhld->bshgd", w, v)
    return out.reshape(B * S, Hq * D).to(state["dtype"])


def _settings(state, rows):
    col = lambda x, t: (x.to(t) if isinstance(x, torch.Tensor) else  # noqa: E731
                        torch.full((rows,), x, dtype=t, device=DEV))[:, None]
    f = lambda k: col(state[k], torch.float32).double()  # noqa: E731  settings are 32-bit values
    return f("temperature"), col(state["top_k"], torch.int64), f("top_p"), f("min_p")


def _plain_sample(state):
    """In 64 bits: a token beside the drawn one is no nearby answer."""
    x = state["logits"].double()
    rows, V = x.shape
    temperature, top_k, top_p, min_p = _settings(state, rows)
    w = torch.exp((x - x.amax(-1, keepdim=True)) / temperature)
    ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)          # ties: the lowest index first
    wr = w.gather(1, order)
    keep = torch.arange(V, device=DEV)[None, :] < torch.where(top_k > 0, top_k, V)
    wr = torch.where(keep, wr, 0.0)
    above = wr.cumsum(-1) - wr                                                   # the mass ranked higher
    keep &= (above <= top_p * wr.sum(-1, keepdim=True)) | (top_p >= 1.0)
    keep &= wr >= min_p
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, wr, 0.0))
    mass = kept.cumsum(-1)
    target = state["random"].double()[:, None] * mass[:, -1:]
    return (mass <= target).sum(-1)


# ── the framework's calls ────────────────────────────────────────────────────

def _package():
    here = os.path.join(os.getcwd(), "csaq-quant_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from csaq import kvcache, sampling
    return kvcache, sampling


def _cache(state):
    """The cache object over the state's buffers, kept with them as a program keeps it."""
    cache = state.get("cache")
    if cache is None:
        kvcache, _ = _package()
        c = state["case"]
        cache = kvcache.QuantizedKVCache.from_buffers(state["k_codes"], state["k_params"], state["v_codes"],
                                                      state["v_params"], bits=c["bits"])
        state["cache"] = cache
        if c["op"] == "attend":
            state["workspace"] = cache.workspace(c["S"], c["Hq"])
    return cache


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "sample": _plain_sample}[op](state)
    if op == "sample":
        if "sample_tokens" not in state:
            state["sample_tokens"] = _package()[1].sample_tokens
        return state["sample_tokens"](state["logits"], state["random"], temperature=state["temperature"],
                                      top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    cache, c = _cache(state), state["case"]
    if op == "write":
        q = cache.write(state["k"], state["v"], state["pos0"], state["cos"], state["sin"], q=state["q"])
        k, v = cache.read(c["start"], c["start"] + c["S"], dtype=state["dtype"])
        return {"q": q, "k": k, "v": v}
    if op == "read":
        k, v = cache.read(0, c["n"], dtype=state["dtype"])
        return {"k": k, "v": v}
    return cache.attend(state["q"], state["pos0"], workspace=state["workspace"])


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["V"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 12 * case["rows"], "flops": 4 * n}
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    stored = Hkv * (D * case["bits"] // 8 + 4 * D // case["group"])  # bytes of one token's keys (or values)
    if case["op"] == "write":
        M = B * case["S"]
        return {"bytes": M * (2 * 2 * Hq * D + 2 * 2 * 2 * Hkv * D + 2 * stored) + 8 * case["S"] * D,
                "flops": M * D * (3 * Hq + 12 * Hkv)}
    if case["op"] == "read":
        return {"bytes": B * case["n"] * 2 * (stored + 2 * Hkv * D), "flops": 2 * 2 * B * case["n"] * Hkv * D}
    S, n = case["S"], case["longest"]
    # ragged lengths are spread evenly from a sixteenth of the longest up to it
    tokens = (n if B == 1 else int(n + (B - 1) * n * 17 / 32)) if case["ragged"] else B * n
    return {"bytes": tokens * 2 * stored + 2 * 2 * B * S * Hq * D, "flops": 4 * tokens * S * Hq * D}


# ── the definition in 64 bits ────────────────────────────────────────────────

def _exact_stored(x, bits, group):
    """What fp64 x (..., D) becomes in the cache."""
    top = 2 ** bits - 1
    y = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    lo = torch.minimum(y.min(-1, keepdim=True).values, torch.zeros((), dtype=torch.float64, device=x.device))
    hi = torch.maximum(y.max(-1, keepdim=True).values, torch.zeros((), dtype=torch.float64, device=x.device))
    step = (hi - lo) / top
    mant, expo = torch.frexp(step)                       # 8 significant bits, upwards
    s = torch.ldexp(torch.ceil(mant * 256.0) / 256.0, expo)
    z = torch.round(-lo / s)
    return ((torch.clamp(torch.round(y / s) + z, 0, top) - z) * s).reshape(x.shape)


def _exact_values(codes, words, bits, group):
    c = codes.to(torch.int64)
    if bits == 4:
        full = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.int64, device=c.device)
        full[..., 0::2], full[..., 1::2] = c % 16, c // 16
        c = full
    w = words.to(torch.int64) % (1 << 32)
    z = (w % 65536 - 0x6400).repeat_interleave(group, dim=-1)
    s = (w // 65536).to(torch.int16).view(torch.bfloat16).double().repeat_interleave(group, dim=-1)
    return (c - z).double() * s


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        rows = case["rows"]
        logits = state["logits"].double().cpu().numpy()
        u = state["random"].double().cpu().numpy()
        one = lambda k, r: (float(state[k][r]) if isinstance(state[k], torch.Tensor)  # noqa: E731
                            else float(np.float32(state[k])))
        out = np.empty(rows, dtype=np.int64)
        for r in range(rows):
            x = logits[r]
            p = np.exp((x - x.max()) / one("temperature", r))
            rank = np.argsort(-x, kind="stable")
            if one("top_k", r) > 0:
                rank = rank[:int(one("top_k", r))]
            mass = np.concatenate([[0.0], np.cumsum(p[rank])])
            if one("top_p", r) < 1.0:
                rank = rank[mass[:-1] <= one("top_p", r) * mass[-1]]
            rank = np.sort(rank[p[rank] >= one("min_p", r)])
            run_up = np.cumsum(p[rank])
            out[r] = rank[np.searchsorted(run_up, u[r] * run_up[-1], side="right")]
        return torch.from_numpy(out).to(DEV)
    B, Hq, Hkv, D, bits, group = (case[k] for k in ("B", "Hq", "Hkv", "D", "bits", "group"))
    if op == "read":
        n = case["n"]
        return {name: _exact_values(state[name + "_codes"][:, :, :n], state[name + "_params"][:, :, :n], bits, group)
                for name in "kv"}
    S = case["S"]
    if op == "write":
        rows = state["cos"][case["start"]:case["start"] + S].double(), state["sin"][case["start"]:case["start"] + S].double()

        def turned(x, h):
            y = x.double().reshape(B, S, h, D)
            other = torch.cat([-y[..., D // 2:], y[..., :D // 2]], dim=-1)
            return y * rows[0][None, :, None] + other * rows[1][None, :, None]

        v = state["v"].double().reshape(B, S, Hkv, D).permute(0, 2, 1, 3)
        return {"q": turned(state["q"], Hq).reshape(B * S, Hq * D),
                "k": _exact_stored(turned(state["k"], Hkv).permute(0, 2, 1, 3), bits, group),
                "v": _exact_stored(v, bits, group)}
    out = torch.empty(B, S, Hq, D, dtype=torch.float64, device=DEV)
    q = state["q"].double().reshape(B, S, Hq, D)
    pos0 = state["pos0"].tolist()
    for b in range(B):
        k = _exact_values(state["k_codes"][b], state["k_params"][b], bits, group)
        v = _exact_values(state["v_codes"][b], state["v_params"][b], bits, group)
        for s in range(S):
            n = pos0[b] + s + 1
            qb = q[b, s].reshape(Hkv, Hq // Hkv, D)
            w = torch.softmax(torch.matmul(qb, k[:, :n].transpose(1, 2)) / math.sqrt(D), dim=-1)
            out[b, s] = torch.matmul(w, v[:, :n]).reshape(Hq, D)
    return out.reshape(B * S, Hq * D)
