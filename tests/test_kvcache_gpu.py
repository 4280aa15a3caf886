"""The quantised KV cache on the GPU: what is written, what is read back and the
attention over it, against plain references (tests/_kv_ref.py).

Codes, scales and zero points are compared bit for bit with the definition in
fp32 numpy operations; reading back is exact up to the one rounding to the
output's type. Attention outputs are compared with 64-bit attention over the
stored values, element by element within

    eps/2 |o|  +  (2^-11 + 2^-12) sum_j w_j |v_j|

eps/2 is the output type's half step. 2^-11 is the half step of the fp16 weights
(relative, each). 2^-12 covers the rest: a score is an fp32 sum of D = 128
products, off by at most 128 2^-24 sum|q k| / sqrt(D), under 2^-13.6 for the
inputs here (sum|q k| / sqrt(D) <= 10), where it changes a weight by that
relative amount and a normaliser by the same; the outputs' own fp32 sums over n
keys are off by sqrt(n) 2^-24 in the usual and n 2^-24 < 2^-13 in the worst case
for n <= 2048.
"""

import math

import numpy as np
import pytest
import torch

import _kv_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYOUTS = [(8, 128, 128), (8, 128, 64), (4, 128, 128), (4, 128, 64), (8, 64, 64), (4, 64, 64)]  # bits, D, group
DTYPES = [torch.bfloat16, torch.float16]


def _tables(n, D):
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2).double() / D))
    f = torch.arange(n).double()[:, None] * inv
    f = torch.cat([f, f], -1)
    return f.cos().float().contiguous(), f.sin().float().contiguous()


def _np(t):
    return t.detach().float().cpu().numpy()


def _cache(B, Hkv, L, D, bits, group):
    from csaq.kvcache import QuantizedKVCache
    return QuantizedKVCache(B, Hkv, L, D, bits=bits, group_size=group, device=DEV)


def _filled(B, Hkv, L, D, bits, group, seed, vscale=1.0):
    """A cache of random keys (with a few large channels) and values."""
    g = torch.Generator().manual_seed(seed)
    c = _cache(B, Hkv, L, D, bits, group)
    gain = torch.ones(D)
    gain[torch.randint(0, D, (2,), generator=g)] = 4.0
    for name, x in (("k", torch.randn(B, Hkv, c.max_len, D, generator=g) * gain * 0.5),
                    ("v", torch.randn(B, Hkv, c.max_len, D, generator=g) * vscale)):
        codes, words = ref.quantise(x.numpy(), bits, group)
        getattr(c, name + "_codes").copy_(torch.from_numpy(ref.pack(codes, bits)))
        getattr(c, name + "_params").copy_(torch.from_numpy(words.view(np.int32)))
    return c


def _values(c, name):
    codes, words = getattr(c, name + "_codes").cpu().numpy(), getattr(c, name + "_params").cpu().numpy().view(np.uint32)
    return torch.from_numpy(ref.values(codes, words, c.bits, c.group_size)).to(DEV)


def _check_attention(out, q, c, pos0, S, scale):
    D = c.head_dim
    want, mag = ref.attention64(q.view(q.shape[0], -1, D), _values(c, "k"), _values(c, "v"), pos0, S, scale)
    got = out.double().view_as(want)
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mag
    tol = tol + torch.finfo(out.dtype).tiny * 2.0 ** -8  # below the type's normal numbers: a step of its subnormals
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()))


# ── writing and reading ──────────────────────────────────────────────────────

@pytest.mark.parametrize("bits,D,group", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,pos", [(1, 1, (0,)), (3, 5, (0, 11, 27)), (2, 33, (7, 0))])
def test_write_is_the_definition(bits, D, group, dtype, B, S, pos):
    Hq, Hkv, L = 6, 2, 64
    g = torch.Generator().manual_seed(bits * 1000 + D + S)
    wide = torch.randn(B * S, (Hq + 2 * Hkv) * D + 16, generator=g).to(dtype).to(DEV)  # a padded fused projection
    q, k, v = wide[:, :Hq * D], wide[:, Hq * D:(Hq + Hkv) * D], wide[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D]
    cos, sin = _tables(L, D)
    c = _cache(B, Hkv, L, D, bits, group)
    before = [t.random_(0, 200).clone() for t in c.buffers()]
    pos0 = torch.tensor(pos, dtype=torch.int32, device=DEV)
    q_rot = c.write(k, v, pos0, cos.to(DEV), sin.to(DEV), q=q)
    p = np.array(pos)[:, None] + np.arange(S)
    cs, sn = cos.numpy()[p][:, :, None], sin.numpy()[p][:, :, None]
    heads = lambda t, h: _np(t).reshape(B, S, h, D)  # noqa: E731
    want_q = torch.from_numpy(ref.rotate(heads(q, Hq), cs, sn)).to(dtype)
    assert torch.equal(q_rot.cpu().view(B, S, Hq, D), want_q)
    for name, x, i in (("k", ref.rotate(heads(k, Hkv), cs, sn), 0), ("v", heads(v, Hkv), 2)):
        codes, words = ref.quantise(x, bits, group)
        want_c, want_w = before[i].cpu().numpy(), before[i + 1].cpu().numpy()
        for b in range(B):
            want_c[b, :, pos[b]:pos[b] + S] = ref.pack(codes[b], bits).swapaxes(0, 1)
            want_w[b, :, pos[b]:pos[b] + S] = words[b].view(np.int32).swapaxes(0, 1)
        assert np.array_equal(getattr(c, name + "_codes").cpu().numpy(), want_c)  # other positions untouched
        assert np.array_equal(getattr(c, name + "_params").cpu().numpy(), want_w)


@pytest.mark.parametrize("bits,D,group", LAYOUTS)
def test_write_edge_values(bits, D, group):
    """Zeros, constants, one sign, the types' extremes, subnormals, NaN and infinities."""
    dtype = torch.bfloat16
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(D), torch.full((D,), 3.0), torch.full((D,), -2.5), torch.rand(D, generator=g) + 1,
            -torch.rand(D, generator=g) - 1, torch.randn(D, generator=g) * 1e38, torch.randn(D, generator=g) * 1e-38,
            torch.randn(D, generator=g) * 1e-40, torch.randn(D, generator=g), torch.randn(D, generator=g),
            torch.randn(D, generator=g), torch.tensor([3.3e38, -3.3e38]).repeat(D // 2)]
    rows[8][3], rows[9][D - 2], rows[10][0] = float("nan"), float("inf"), float("-inf")
    x = torch.stack(rows).to(dtype)
    c = _cache(len(rows), 1, 16, D, bits, group)
    c.write(x.to(DEV), x.to(DEV), torch.full((len(rows),), 9, dtype=torch.int32, device=DEV))
    codes, words = ref.quantise(x.float().numpy(), bits, group)
    for name in "kv":
        assert np.array_equal(getattr(c, name + "_codes").cpu().numpy()[:, 0, 9], ref.pack(codes, bits))
        assert np.array_equal(getattr(c, name + "_params").cpu().numpy()[:, 0, 9], words.view(np.int32))
    back = c.read(9, 10, dtype=torch.float32)[0][:, 0, 0].cpu().double()
    xd = x.double()
    for r in range(8):  # the documented bound
        gr = xd[r].view(-1, group)
        span = gr.amax(-1).clamp(min=0) - gr.amin(-1).clamp(max=0)
        s = (1.01 * span / (2 ** bits - 1)).clamp(min=2.0 ** -126)
        assert ((back[r].view(-1, group) - gr).abs() <= 1.01 * s[:, None]).all()
    for r, bad in ((8, 3), (9, D - 2), (10, 0)):
        grp = back[r].view(-1, group)
        assert grp[bad // group].isnan().all()
        assert grp.isnan().all(-1).sum() == 1


@pytest.mark.parametrize("bits,D,group", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_between_two_codes(bits, D, group, dtype):
    """Quotients on and right beside the middle between two codes, for many scales: the
    neighbours of (i + 1/2) s in dtype, s the group's scale."""
    n, rows = 2 ** bits - 1, 600
    g = torch.Generator().manual_seed(17)
    s = torch.exp2(torch.rand(rows, 1, generator=g) * 8 - 8).bfloat16().float()
    low = torch.randint(0, n, (rows, 1), generator=g).float()  # codes from -low to n - low
    x = (torch.randint(0, n, (rows, D), generator=g) - low + 0.5).clamp(max=n - 0.5) * s
    x = x.to(dtype)
    step = torch.randint(-1, 2, x.shape, generator=g, dtype=torch.int16)
    x = (x.view(torch.int16) + step).view(dtype)
    x[:, ::group], x[:, 1::group] = (-low * s).to(dtype), ((n - low) * s).to(dtype)
    c = _cache(rows, 1, 16, D, bits, group)
    c.write(x.to(DEV), x.to(DEV), torch.zeros(rows, dtype=torch.int32, device=DEV))
    codes, words = ref.quantise(x.float().numpy(), bits, group)
    assert np.array_equal(c.k_codes.cpu().numpy()[:, 0, 0], ref.pack(codes, bits))
    assert np.array_equal(c.k_params.cpu().numpy()[:, 0, 0], words.view(np.int32))


def test_write_skips_positions_outside():
    """Before 0, behind the cache and behind the tables nothing is stored; the
    queries there pass unrotated."""
    B, S, Hq, Hkv, D, L = 3, 4, 2, 1, 64, 32
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(B * S, h * D, generator=g).to(torch.bfloat16).to(DEV) for h in (Hq, Hkv, Hkv))
    cos, sin = _tables(24, D)
    c = _cache(B, Hkv, L, D, 8, 64)
    before = [t.random_(0, 99).clone() for t in c.buffers()]
    pos0 = torch.tensor([-2, 22, 30], dtype=torch.int32, device=DEV)
    q_rot = c.write(k, v, pos0, cos.to(DEV), sin.to(DEV), q=q).view(B, S, Hq, D)
    stored = {0: [0, 1], 1: [22, 23], 2: []}
    for t, old in zip(c.buffers(), before):
        for b in range(B):
            changed = (t[b] != old[b]).any(-1).any(0).nonzero().flatten().tolist()
            assert set(changed) <= set(stored[b])
    assert torch.equal(q_rot[2], q.view(B, S, Hq, D)[2]) and torch.equal(q_rot[0, :2], q.view(B, S, Hq, D)[0, :2])
    # without tables positions up to the cache's end are stored
    c.write(k, v, pos0)
    assert (c.v_codes[2, :, 30:] != before[2][2, :, 30:]).any()


@pytest.mark.parametrize("bits,D,group", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_read_is_exact(bits, D, group, dtype):
    c = _filled(2, 3, 48, D, bits, group, seed=D + bits)
    for start, end in ((0, 48), (5, 6), (17, 40), (8, 8)):
        k, v = c.read(start, end, dtype=dtype)
        for name, t in (("k", k), ("v", v)):
            want = _values(c, name)[:, :, start:end].float().to(dtype)  # fp32 holds the values exactly
            assert t.shape == want.shape and torch.equal(t, want)
    out = (torch.empty(2, 3, 4, D, dtype=dtype, device=DEV), torch.empty(2, 3, 4, D, dtype=dtype, device=DEV))
    assert c.read(1, 5, dtype=dtype, out=out)[0] is out[0]
    assert torch.equal(out[1], c.read(0, 5, dtype=dtype)[1][:, :, 1:])


# ── attention ────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("bits,D,group", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_lengths(bits, D, group, dtype):
    """One to a few hundred keys around every tile and chunk border, in one batch."""
    lens = [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 143, 255, 256, 257, 300, 400]
    B, Hq, Hkv, L = len(lens), 8, 2, 400
    c = _filled(B, Hkv, L, D, bits, group, seed=3)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(B, Hq * D, generator=g).to(dtype).to(DEV)
    pos0 = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV)
    out = c.attend(q, pos0)
    _check_attention(out, q, c, pos0.tolist(), 1, 1 / math.sqrt(D))


@pytest.mark.parametrize("Hq,Hkv,S", [(1, 1, 1), (7, 1, 1), (3, 3, 2), (8, 1, 1), (16, 2, 2), (14, 2, 3), (32, 8, 5),
                                      (16, 16, 9), (8, 1, 4), (4, 2, 31), (12, 1, 7)])
@pytest.mark.parametrize("bits,D,group", [(8, 128, 128), (4, 128, 64), (4, 64, 64)])
def test_attention_heads_and_tokens(Hq, Hkv, S, bits, D, group):
    """Group sizes from 1 to 12 and several tokens a step: one to several blocks of query rows."""
    B, L = 3, 700
    c = _filled(B, Hkv, L, D, bits, group, seed=Hq + S)
    g = torch.Generator().manual_seed(S)
    q = torch.randn(B * S, Hq * D, generator=g).to(torch.bfloat16).to(DEV)
    pos0 = torch.tensor([0, 123, c.max_len - S], dtype=torch.int32, device=DEV)
    out = c.attend(q, pos0, scale=0.11)
    _check_attention(out, q, c, pos0.tolist(), S, 0.11)


def test_attention_rows_without_keys():
    """Tokens before position 0 see nothing and give zeros, tokens behind the cache
    see all of it; unused sequences of a batch are all zeros."""
    B, S, Hq, Hkv, D = 4, 4, 4, 2, 128
    c = _filled(B, Hkv, 160, D, 8, 128, seed=9)
    q = torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(2)).to(torch.float16).to(DEV)
    pos0 = torch.tensor([-4, -2, 158, 2_000_000_000], dtype=torch.int32, device=DEV)
    out = torch.full((B * S, Hq * D), float("nan"), dtype=torch.float16, device=DEV)
    c.attend(q, pos0, out=out)
    _check_attention(out, q, c, pos0.tolist(), S, 1 / math.sqrt(D))
    assert (out[:4] == 0).all() and (out[4:6] == 0).all() and (out[6:8] != 0).any()
    pos0.fill_(-2_000_000_000)
    assert (c.attend(q, pos0) == 0).all()


@pytest.mark.parametrize("bits,D,group", LAYOUTS)
def test_attention_ignores_what_is_behind(bits, D, group):
    """Codes and parameters behind the last visible key may be anything, NaN scales
    and zero points that are no numbers among them."""
    B, S, Hq, Hkv = 3, 2, 4, 2
    c = _filled(B, Hkv, 320, D, bits, group, seed=11)
    q = torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    pos0 = torch.tensor([0, 18, 200], dtype=torch.int32, device=DEV)
    clean = c.attend(q, pos0)
    for b, p in enumerate(pos0.tolist()):
        for t in (c.k_params, c.v_params):
            t[b, :, p + S:] = torch.tensor(0x7FC07E01, dtype=torch.int32)
        for t in (c.k_codes, c.v_codes):
            t[b, :, p + S:] = 255
    assert torch.equal(c.attend(q, pos0), clean)
    # the token before it must not see the last key either, whatever that holds
    c.v_params[:, :, :] = torch.where(torch.arange(320, device=DEV)[None, None, :, None] ==
                                      (pos0[:, None, None, None] + 1), 0x7FC06400, c.v_params)
    out = c.attend(q, pos0).view(B, S, -1)
    assert torch.equal(out[:, 0], clean.view(B, S, -1)[:, 0]) and out[:, 1].isnan().all()


@pytest.mark.parametrize("what", ["q", "k", "v"])
def test_attention_passes_nan_on(what):
    """A NaN among what a row sees makes that row NaN and no other."""
    B, Hq, Hkv, D = 2, 4, 2, 128
    c = _filled(B, Hkv, 64, D, 8, 128, seed=12)
    q = torch.randn(B, Hq * D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    pos0 = torch.tensor([40, 50], dtype=torch.int32, device=DEV)
    clean = c.attend(q, pos0).view(B, Hq, D)
    if what == "q":
        q[1, 2 * D + 5] = float("nan")
        hit = torch.tensor([[0, 0, 0, 0], [0, 0, 1, 0]], dtype=torch.bool, device=DEV)
    else:
        getattr(c, what + "_params")[1, 1, 7] = 0x7FC06400
        hit = torch.tensor([[0, 0, 0, 0], [0, 0, 1, 1]], dtype=torch.bool, device=DEV)
    out = c.attend(q, pos0).view(B, Hq, D)
    assert out[hit].isnan().all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("vscale", [1e-12, 1e-4, 3e4])
@pytest.mark.parametrize("qscale", [1e-4, 30.0])
def test_attention_scales(vscale, qscale):
    """Very small and very large values, flat and one-hot weights (bf16)."""
    B, Hq, Hkv, D = 2, 4, 2, 128
    c = _filled(B, Hkv, 500, D, 8, 128, seed=13, vscale=vscale)
    # with scores of up to +-300 a relative error of 2^-24 in a score counts as much in a weight
    q = (torch.randn(B, Hq * D, generator=torch.Generator().manual_seed(5)) * qscale).to(torch.bfloat16).to(DEV)
    q = (q.float() * 2.0 ** torch.randint(-4, 1, (B, 1), generator=torch.Generator().manual_seed(6)).to(DEV)).to(q.dtype)
    pos0 = torch.tensor([499, 333], dtype=torch.int32, device=DEV)
    want, mag = ref.attention64(q.view(B, Hq, D), _values(c, "k"), _values(c, "v"), pos0.tolist(), 1, D ** -0.5)
    out = c.attend(q, pos0).double().view_as(want)
    dots = torch.einsum("bhgd,bhld->bhgl", q.double().view(B, Hkv, 2, D).abs(), _values(c, "k").abs()).amax() / D ** 0.5
    # as in the module's comment, with this test's own bound of the scores' error
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13 + 2 * 128 * 2.0 ** -24 * float(dots)) * mag
    assert ((out - want).abs() <= tol).all()


def test_attention_many_equal_weights_beside_a_large_one():
    """One key outweighs each of 32767 others by 2^20 and more: together they still
    count. The many heads (all alike) make the chunks as long as the cache."""
    Hkv, D, L = 1184, 64, 32768
    c = _cache(1, Hkv, L, D, 8, 64)
    x = torch.zeros(L, D)
    x[:, 0] = -16.0          # score of the many; the one has 0
    x[5, 0] = 0.0
    y = torch.ones(L, D)
    y[5] = -1.0
    for name, t in (("k", x), ("v", y)):
        codes, words = ref.quantise(t.numpy(), 8, 64)
        getattr(c, name + "_codes").copy_(torch.from_numpy(ref.pack(codes, 8)).to(DEV)[None, None])
        getattr(c, name + "_params").copy_(torch.from_numpy(words.view(np.int32)).to(DEV)[None, None])
    q = torch.zeros(2, D)
    q[0, 0], q[1, 0] = 1.0, 0.9
    q = q.to(torch.float16).to(DEV)
    pos0 = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    out = c.attend(q.view(1, 2 * D).repeat(1, Hkv), pos0, scale=1.0).view(Hkv, 2, D)
    assert torch.equal(out, out[:1].expand_as(out))
    one = type(c).from_buffers(*(t[:, :1].contiguous() for t in c.buffers()), bits=8)
    want, mag = ref.attention64(q.view(1, 2, D), _values(one, "k"), _values(one, "v"), [L - 1], 1, 1.0)
    # in the warp that holds the large weight as 2^7 the many of row 0 are near 2^-16, a fp16
    # subnormal with a half step of 2^-25: 2^-9 of each, and their sum is 2^15 2^-23
    tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mag + 2.0 ** -9 * 2.0 ** -8
    got = out[:1].double()
    assert ((got - want).abs() <= tol).all()
    assert float((got[0, 1] + 1).abs().min()) > 0.02  # 32767 e^-14.4 is 0.018, twice that


def test_attention_offsets_past_32_bits():
    """A cache of over 4 GiB of codes: the last head of the last sequence."""
    B, Hkv, D, L = 1, 34, 128, 1 << 20
    c = _cache(B, Hkv, L, D, 8, 128)
    assert c.k_codes.numel() > 1 << 32
    g = torch.Generator().manual_seed(8)
    n = 1500
    pos0 = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(n, Hkv * D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    c.write(k, v, pos0 - (n - 1))
    q = torch.randn(1, Hkv * D, generator=g).to(torch.bfloat16).to(DEV)
    out = c.attend(q, pos0).view(Hkv, D)
    kk, vv = c.read(L - n, L, dtype=torch.float32)
    # the L - n zero keys have score 0 and value 0
    for h in (0, Hkv - 1):
        s = (kk[0, h].double() @ q.double().view(Hkv, D)[h]) * D ** -0.5
        w = s.exp() / (s.exp().sum() + (L - n))
        want, mag = w @ vv[0, h].double(), w @ vv[0, h].double().abs()
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mag
        assert ((out[h].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("bits,D,group", [(8, 128, 128), (4, 128, 64), (4, 64, 64)])
def test_attention_independent_of_the_step(bits, D, group):
    """A token's result is bitwise the same alone, among more tokens (one or several
    row blocks) and beside other sequences."""
    Hq, Hkv, L, S = 16, 2, 900, 5
    c = _filled(2, Hkv, L, D, bits, group, seed=21)
    q = torch.randn(2 * S, Hq * D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(DEV)
    pos0 = torch.tensor([253, 700], dtype=torch.int32, device=DEV)
    together = c.attend(q, pos0).view(2, S, -1)
    for s in range(S):
        alone = c.attend(q.view(2, S, -1)[:, s].contiguous(), pos0 + s)
        assert torch.equal(alone, together[:, s])
    other = c.attend(q, torch.tensor([253, 3], dtype=torch.int32, device=DEV)).view(2, S, -1)
    assert torch.equal(other[0], together[0])


@pytest.mark.parametrize("bits,D,group", [(8, 128, 128), (4, 128, 64), (4, 64, 64), (8, 64, 64)])
@pytest.mark.parametrize("S", [2, 3, 5])
def test_attention_independent_of_the_row_blocks(bits, D, group, S):
    """The same where there are CTAs enough for blocks of 16 and 24 rows: 64 KV heads
    of 8 query heads, 16, 24 and 40 rows each, against the 8 of a token alone."""
    B, Hq, Hkv, L = 8, 64, 8, 900
    c = _filled(B, Hkv, L, D, bits, group, seed=22)
    q = 3 * torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(DEV)
    pos0 = torch.tensor([0, 1, 15, 130, 511, 513, 700, 894], dtype=torch.int32, device=DEV)
    together = c.attend(q, pos0).view(B, S, -1)
    for s in range(S):
        assert torch.equal(c.attend(q.view(B, S, -1)[:, s].contiguous(), pos0 + s), together[:, s])


def test_attention_strides_workspaces_and_repeats():
    """Padded rows of q and out (the padding stays), an own workspace used over and
    over with other lengths and token counts, equal bits."""
    B, Hq, Hkv, D, L = 2, 8, 2, 128, 2000
    c = _filled(B, Hkv, L, D, 8, 64, seed=31)
    ws = c.workspace(4, Hq)
    g = torch.Generator().manual_seed(7)
    for S, pos in ((4, (1990, 3)), (1, (1500, 1999)), (2, (0, 700)), (4, (1990, 3))):
        pos0 = torch.tensor(pos, dtype=torch.int32, device=DEV)
        wide = torch.randn(B * S, Hq * D + 24, generator=g).to(torch.bfloat16).to(DEV)
        q = wide[:, :Hq * D]
        buf = torch.full((B * S, Hq * D + 6), 7.0, dtype=torch.bfloat16, device=DEV)
        out = c.attend(q, pos0, out=buf[:, :Hq * D], workspace=ws)
        assert (buf[:, Hq * D:] == 7).all()
        assert torch.equal(out, c.attend(q.contiguous(), pos0))
        _check_attention(out, q.contiguous(), c, pos, S, D ** -0.5)
        odd = torch.empty(B * S * Hq * D + 3, dtype=torch.bfloat16, device=DEV)[3:].view(B * S, Hq * D).copy_(q)
        assert torch.equal(c.attend(odd, pos0), out)  # rows the kernel cannot read in place are copied
    big = _cache(1, 2, 1 << 20, 128, 4, 64)  # chunks that meet in global memory
    with pytest.raises(ValueError, match="workspace"):
        big.attend(torch.zeros(5, 1024, dtype=torch.bfloat16, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                   workspace=big.workspace(4, 8))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("Hkv", [4, 24, 80])
def test_scratch_that_is_not_needed(bits, Hkv):
    """Scratch sized for either width of codes changes nothing where a head's chunks
    meet in a cluster; 24 heads of a long 4-bit cache leave partials."""
    D, L, n = 64, 20480, 700
    c = _cache(1, Hkv, L, D, bits, 64)
    g = torch.Generator().manual_seed(31)
    k, v, q = (torch.randn(m, Hkv * D, generator=g).to(torch.float16).to(DEV) for m in (n, n, 1))
    pos0 = torch.tensor([L - n], dtype=torch.int32, device=DEV)
    c.write(k, v, pos0)
    at = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    from csaq.kvcache import KVWorkspace
    out = c.attend(q, at, workspace=KVWorkspace(torch.zeros(Hkv * 600 * (D + 2), device=DEV))).view(Hkv, D)
    assert torch.equal(out, c.attend(q, at).view(Hkv, D))
    kk, vv = (t[0, :, L - n:].double() for t in c.read(0, L, dtype=torch.float32))
    s = torch.einsum("hd,hnd->hn", q.double().view(Hkv, D), kk) * D ** -0.5
    w = s.exp() / (s.exp().sum(1, keepdim=True) + (L - n))  # the zero keys have score 0 and value 0
    want, mag = torch.einsum("hn,hnd->hd", w, vv), torch.einsum("hn,hnd->hd", w, vv.abs())
    # roundings of the output (2^-25 below the normal numbers), of each weight times its
    # value's scale, and the scores' own
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -12) * mag
    assert ((out.double() - want).abs() <= tol).all()


def test_decode_loop_captured():
    """Prompt, then steps of write + attend as one captured graph, against 64-bit
    attention over everything written; another stream with its own workspace
    runs the same steps eagerly and gives the same bits."""
    B, Hq, Hkv, D, P, steps = 2, 8, 2, 128, 150, 6
    g = torch.Generator().manual_seed(17)
    dt = torch.bfloat16
    cos, sin = (t.to(DEV) for t in _tables(256, D))
    rows = (Hq + 2 * Hkv) * D
    prompt = torch.randn(B * P, rows, generator=g).to(dt).to(DEV)
    news = torch.randn(steps, B, rows, generator=g).to(dt).to(DEV)
    split = lambda x: (x[:, :Hq * D], x[:, Hq * D:(Hq + Hkv) * D], x[:, (Hq + Hkv) * D:])  # noqa: E731

    def start():
        c = _cache(B, Hkv, 256, D, 8, 128)
        q, k, v = split(prompt)
        pos0 = torch.zeros(B, dtype=torch.int32, device=DEV)
        c.write(k, v, pos0, cos, sin)
        return c, pos0.fill_(P), c.workspace(1, Hq)

    def step(c, x, pos0, ws, q_out, out):
        q, k, v = split(x)
        c.write(k, v, pos0, cos, sin, q=q, q_out=q_out)
        c.attend(q_out, pos0, out=out, workspace=ws)
        pos0.add_(1)

    bufs = lambda: (torch.empty(B, Hq * D, dtype=dt, device=DEV), torch.empty(B, Hq * D, dtype=dt, device=DEV))  # noqa: E731
    c1, pos1, ws1 = start()
    q1, o1 = bufs()
    x = news[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c1, x, pos1, ws1, q1, o1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c1, x, pos1, ws1, q1, o1)
    pos1.fill_(P)
    c2, pos2, ws2 = start()
    q2, o2 = bufs()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for i in range(steps):
        x.copy_(news[i])
        graph.replay()
        with torch.cuda.stream(other):
            step(c2, news[i], pos2, ws2, q2, o2)
        torch.cuda.synchronize()
        assert torch.equal(o1, o2)
        _check_attention(o1, q1, c1, [P + i] * B, 1, D ** -0.5)
    assert all(torch.equal(a, b) for a, b in zip(c1.buffers(), c2.buffers()))


def test_refusals_on_the_device():
    c = _cache(2, 2, 32, 128, 8, 128)
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
    pos = z(2, t=torch.int32)
    k = z(4, 256)
    cos = z(32, 128, t=torch.float32)
    for args, kw, exc in (((k.float(), k.float(), pos), {}, TypeError), ((z(3, 256), k, pos), {}, ValueError),
                          ((k, z(2, 256), pos), {}, ValueError), ((k, z(4, 128), pos), {}, ValueError),
                          ((k, k.half(), pos), {}, ValueError), ((k, k, pos.long()), {}, ValueError),
                          ((k, k, z(3, t=torch.int32)), {}, ValueError), ((k, k, pos, cos), {}, ValueError),
                          ((k, k, pos, cos[:, :64], cos[:, :64]), {}, ValueError),
                          ((k, k, pos, cos.half(), cos.half()), {}, ValueError),
                          ((k, k, pos), dict(q=k), ValueError), ((k, k, pos, cos, cos), dict(q=z(4, 200)), ValueError),
                          ((k, k, pos, cos, cos), dict(q=z(2, 256)), ValueError),
                          ((k, k, pos, cos, cos), dict(q_out=z(4, 256)), ValueError),
                          ((k.cpu(), k.cpu(), pos), {}, RuntimeError)):
        with pytest.raises(exc):
            c.write(*args, **kw)
    for args, kw, exc in (((z(4, 300), pos), {}, ValueError), ((z(4, 128), pos), {}, ValueError),
                          ((z(4, 256, t=torch.float32), pos), {}, TypeError), ((k, pos.cpu()), {}, ValueError),
                          ((k, pos), dict(out=z(4, 128)), ValueError), ((k, pos), dict(out=z(4, 256).half()), ValueError)):
        with pytest.raises(exc):
            c.attend(*args, **kw)
    with pytest.raises(TypeError):
        c.read(0, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        c.read(0, 4, out=(z(2, 2, 4, 128), z(2, 2, 3, 128)))
