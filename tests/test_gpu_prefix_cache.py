"""Shared-prefix attention, key weights, the weighted decode step and cache eviction (hk_attn_prefix.hip, hk_cache.hip) against
plain 64-bit restatements on the same inputs.

Tolerances are element-wise and come from the roundings alone.  With A = sum_j p_j |v_j| (p normalised), the output of an attention
row is off by at most
    2^-8 A      P enters the matrix instruction in bf16 (half a step relative to each p_j),
    2^-8 |o|    the output's own rounding,
    2 d A       scores: d = ln 2 * hd * 2^-24 * max |q| . |k| bounds the relative error of every p_j before normalisation,
and a weight sum of n terms by (2 d + (n + 128) 2^-24) of itself (exp2, the row's log2 sum below 2^6, the additions)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from hawkeye_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOG2E = 1.4426950408889634
NAN, INF = float("nan"), float("inf")


def _rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DEV).to(dtype)


def _bias(kind, B, n, seed, value=-1.0e4):
    """None | 'left': rows left-padded to different lengths | 'holes' | 'add': finite biases and holes | 'all': the last row empty"""
    if kind is None:
        return None
    g = torch.Generator(device="cpu").manual_seed(seed)
    if kind == "left":
        valid = torch.randint(1, n + 1, (B,), generator=g)
        gone = torch.arange(n)[None] < (n - valid)[:, None]
    else:
        gone = torch.rand((B, n), generator=g) < 0.4
        if kind == "all":
            gone[-1] = True
    b = torch.zeros((B, n))
    if kind == "add":
        b = torch.randn((B, n), generator=g) * 2
    b[gone] = value
    return b.to(DEV)


def _softmax(q, ks, biases, nq):
    """q [B,H,Nq,hd] double, ks: [B,H,n,hd] double pieces; biases the same in [B,H,1,n] (or None); the LAST piece is causal."""
    parts = []
    for i, (k, b) in enumerate(zip(ks, biases)):
        s = (q @ k.transpose(2, 3)) * math.log(2.0)
        if b is not None:
            s = torch.where(b <= -1.0e4, torch.full_like(s, -INF), s + b)
        if i == len(ks) - 1 and nq is not None:
            n = k.shape[2]
            s = s.masked_fill(torch.arange(n, device=s.device)[None] > torch.arange(nq, device=s.device)[:, None] + n - nq, -INF)
        parts.append(s)
    s = torch.cat(parts, -1)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -INF, torch.zeros_like(top), top))
    tot = e.sum(-1, keepdim=True)
    return e / torch.where(tot == 0, torch.ones_like(tot), tot)


def _d(q, ks, hd):
    """The score error bound d, for the whole problem."""
    big = max(float((q.abs() @ k.abs().nan_to_num(0.0).transpose(2, 3)).max()) if k.shape[2] else 0.0 for k in ks)
    return math.log(2.0) * hd * 2.0 ** -24 * big


def _h(t):
    return t.double().transpose(1, 2)         # [B,N,H,hd] -> [B,H,N,hd]


def _ref_prefix(q, kp, vp, k, v, bias):
    B, nq, H, hd = q.shape
    qd, ks = _h(q), [_h(kp[None]).expand(B, -1, -1, -1), _h(k)]
    vs = torch.cat([_h(vp[None]).expand(B, -1, -1, -1), _h(v)], 2)
    gone = None if bias is None else (bias <= -1.0e4)[:, None, :, None]
    if gone is not None:                      # what stands in a removed row does not count
        ks[1] = ks[1].masked_fill(gone, 0.0)
        vs = torch.cat([vs[:, :, :kp.shape[0]], vs[:, :, kp.shape[0]:].masked_fill(gone, 0.0)], 2)
    p = _softmax(qd, ks, [None, None if bias is None else bias.double()[:, None, None]], nq)
    out, A = p @ vs, p @ vs.abs()
    tol = 2.0 ** -8 * (A + out.abs()) + 2 * _d(qd, ks, hd) * A + 1e-37
    return out.transpose(1, 2), tol.transpose(1, 2)


def _near(got, ref, tol):
    assert got.shape == ref.shape
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - ref).abs() / tol).nan_to_num(INF).max()):.3g} times the bound"


PREFIX = [  # B, Nq, P, Nk, H, hd, bias
    (1, 1, 0, 1, 1, 64, None), (1, 1, 1, 1, 2, 128, None), (3, 1, 33, 5, 2, 128, None), (2, 1, 0, 40, 3, 64, "all"), (16, 1, 500, 70, 32, 128, "left"),
    (17, 1, 64, 1, 5, 64, None), (40, 1, 129, 33, 3, 128, "left"), (64, 1, 1000, 100, 2, 128, "add"), (70, 1, 31, 32, 1, 64, "holes"),
    (40, 1, 1100, 1100, 32, 128, None), (1, 1, 5000, 3000, 2, 128, "holes"), (4, 1, 352, 20, 32, 128, None),
    (2, 5, 0, 9, 2, 128, "all"), (5, 3, 777, 130, 12, 64, "add"), (1, 16, 100, 16, 2, 128, None), (3, 17, 64, 64, 2, 64, "holes"),
    (7, 37, 201, 37, 4, 128, "left"), (2, 130, 100, 200, 2, 128, "holes"), (1, 64, 1, 64, 1, 64, None), (2, 257, 300, 257, 3, 128, "left"),
    (1, 129, 0, 129, 2, 64, "all"), (3, 200, 1030, 700, 2, 64, "add"), (2, 512, 1400, 512, 2, 128, None), (9, 100, 65, 100, 2, 128, "left"),
    (16, 5, 700, 60, 3, 128, "left"), (33, 3, 129, 40, 2, 64, "holes"), (4, 32, 2000, 32, 8, 128, None), (1, 64, 0, 5000, 1, 64, "add"),
    (1, 100, 0, 3000, 2, 128, "left"), (40, 64, 64, 64, 32, 64, "all"), (1, 33, 4097, 1100, 1, 128, "holes"),
]


@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", PREFIX)
def test_prefix_attention_matches_its_definition(B, Nq, P, Nk, H, hd, kind):
    qs = 1.5 * hd ** -0.5 * LOG2E
    q = _rand((B, Nq, 3, H, hd), 1, qs)[:, :, 1]                         # a strided view, as the projection leaves it
    kp, vp = _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    rows = Nk + 3
    k, v = _rand((B, rows, H, hd), 4), _rand((B, rows, H, hd), 5)
    k[:, Nk:], v[:, Nk:] = NAN, NAN                                      # cache rows not filled yet
    bias = _bias(kind, B, Nk, 6, -INF if kind == "holes" else -1.0e4)
    if bias is not None:
        gone = bias <= -1.0e4
        k[:, :Nk][gone], v[:, :Nk][gone] = NAN, INF                      # removed rows may hold anything
    out = torch.full((B, Nq + 1, H, hd), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ops.prefix_attention(q, kp, vp, k[:, :Nk], v[:, :Nk], key_bias=bias, out=out[:, :Nq])
    ref, tol = _ref_prefix(q, kp, vp, k[:, :Nk], v[:, :Nk], bias)
    _near(got, ref, tol)
    assert bool((out[:, Nq:] == 7.0).all())
    again = ops.prefix_attention(q, kp, vp, k[:, :Nk], v[:, :Nk], key_bias=bias)
    assert torch.equal(again, got)
    if kind == "all" and P == 0:
        assert bool((got[-1] == 0).all())


@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", [           # one workgroup for prefix and own keys: two groups of waves, and (last three) one
    (2, 130, 300, 130, 6, 128, "left"), (1, 512, 333, 512, 5, 64, "add"), (3, 200, 0, 450, 4, 128, "all"), (1, 257, 0, 460, 8, 128, "holes"),
    (4, 64, 385, 64, 16, 64, None), (2, 385, 0, 385, 3, 128, "left"), (3, 40, 100, 41, 90, 64, "left"), (2, 150, 200, 150, 70, 128, "add"), (5, 33, 64, 33, 60, 128, "all")])
def test_prefix_attention_in_one_launch_of_row_blocks(B, Nq, P, Nk, H, hd, kind):
    test_prefix_attention_matches_its_definition(B, Nq, P, Nk, H, hd, kind)


@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", [           # many sequences with few own keys: a wave per (sequence, head)
    (33, 1, 500, 61, 32, 64, "left"), (130, 1, 400, 20, 9, 128, "add"), (70, 3, 300, 33, 15, 64, "holes"), (40, 20, 200, 70, 30, 128, "all"),
    (257, 1, 33, 96, 5, 128, "left"), (1030, 1, 700, 1, 1, 64, None), (26, 1, 2100, 97, 40, 128, "left"), (128, 2, 6000, 31, 9, 128, "holes")])
def test_prefix_attention_of_many_short_sequences(B, Nq, P, Nk, H, hd, kind):
    test_prefix_attention_matches_its_definition(B, Nq, P, Nk, H, hd, kind)


def test_prefix_attention_large_scores_and_late_maximum():
    """Scores that grow along the keys by far more than the lazily moved maximum's 8 bits, up to 2^10 apart."""
    B, P, Nk, H, hd = 3, 400, 50, 2, 128
    q, kp, vp = _rand((B, 1, H, hd), 1, 1.0), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    kp = (kp.float() * torch.linspace(0.1, 30, P, device=DEV)[:, None, None]).to(torch.bfloat16)
    k, v = _rand((B, Nk, H, hd), 4, 5.0), _rand((B, Nk, H, hd), 5)
    got = ops.prefix_attention(q, kp, vp, k, v)
    ref, tol = _ref_prefix(q, kp, vp, k, v, None)
    _near(got, ref, tol)


def _ref_weights(q, k, bias, causal):
    """softmax weights [B,H,Nq,Nk] in 64 bits and d; bias [B,n] or [B,H,n]"""
    hd = q.shape[3]
    qd, kd = _h(q), _h(k)
    b = None
    if bias is not None:
        b = bias.double()[:, None, None] if bias.dim() == 2 else bias.double()[:, :, None]
        kd = kd.masked_fill((b <= -1.0e4).transpose(2, 3), 0.0)
    return _softmax(qd, [kd], [b], q.shape[1] if causal else None), _d(qd, [kd], hd)


@pytest.mark.parametrize("B,n,H,hd,kind", [(1, 1, 1, 64, None), (2, 2, 2, 128, None), (1, 353, 32, 128, None), (16, 300, 4, 128, "left"), (3, 2500, 2, 64, "add"),
                                           (2, 127, 3, 128, "all"), (5, 1029, 2, 128, "head"), (1, 70000, 1, 64, None), (40, 33, 32, 64, "holes")])
def test_decode_attn_weights_matches_its_definition(B, n, H, hd, kind):
    rows = n + 5
    q = _rand((B, H * hd), 1, 1.5 * hd ** -0.5 * LOG2E)
    k, v = _rand((B, rows, H * hd), 2), _rand((B, rows, H * hd), 3)
    k[:, n:], v[:, n:] = NAN, NAN
    bias = _bias("holes", B * H, n, 4).view(B, H, n) if kind == "head" else _bias(kind, B, n, 4)
    if bias is not None and bias.dim() == 2:
        k[:, :n][bias <= -1.0e4], v[:, :n][bias <= -1.0e4] = NAN, NAN
    w = _rand((B, H, rows), 5, 1.0, torch.float32).abs()
    wo = torch.full_like(w, 7.0)
    out = ops.decode_attn_weights(q, k, v, n, H, hd, w, key_bias=bias, weight_out=wo)
    kk, vv = k[:, :n].view(B, n, H, hd), v[:, :n].view(B, n, H, hd)
    p, d = _ref_weights(q.view(B, 1, H, hd), kk, bias, False)
    vd = _h(vv)
    if bias is not None:
        vd = vd.masked_fill((bias <= -1.0e4)[..., None] if bias.dim() == 3 else (bias <= -1.0e4)[:, None, :, None], 0.0)
    ref, A = (p @ vd)[:, :, 0], (p @ vd.abs())[:, :, 0]
    _near(out.view(B, H, hd), ref, 2.0 ** -8 * (A + ref.abs()) + 2 * d * A + 1e-37)
    pw = p[:, :, 0]
    _near(wo[..., :n], w[..., :n].double() + pw, pw * (2 * d + 129 * 2.0 ** -24) + 2.0 ** -23 * (w[..., :n].double() + pw) + 1e-37)
    assert bool((wo[..., n:] == 7.0).all())
    inplace = w.clone()
    assert torch.equal(ops.decode_attn_weights(q, k, v, n, H, hd, inplace, key_bias=bias), out)
    assert torch.equal(inplace[..., :n], wo[..., :n]) and torch.equal(inplace[..., n:], w[..., n:])
    fresh = torch.full_like(w, 7.0)
    ops.decode_attn_weights(q, k, v, n, H, hd, None, key_bias=bias, weight_out=fresh)
    _near(fresh[..., :n], pw, pw * (2 * d + 130 * 2.0 ** -24) + 1e-37)


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [
    (1, 1, 1, 1, 64, True, None), (1, 352, 352, 4, 128, True, None), (2, 333, 333, 3, 64, True, "left"), (1, 32, 500, 2, 128, True, "holes"),
    (2, 65, 64, 2, 128, False, None), (1, 1, 700, 2, 64, True, "add"), (3, 129, 130, 2, 128, True, "all"), (1, 1500, 1500, 2, 128, True, None),
    (2, 200, 31, 2, 64, False, "add"), (1, 40, 40, 1, 128, False, "all")])
def test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind):
    n = max(Nq, Nk)
    qkv = _rand((B, n, 3, H, hd), 1)
    qkv[:, :, 0] *= 1.5 * hd ** -0.5 * LOG2E
    q, k = qkv[:, n - Nq:, 0], qkv[:, :Nk, 1]
    bias = _bias(kind, B, Nk, 2, -INF if kind == "holes" else -1.0e4)
    if bias is not None:
        k[bias <= -1.0e4] = NAN
    got = ops.attn_key_weights(q, k, key_bias=bias, causal=causal)
    p, d = _ref_weights(q, k, bias, causal)
    ref = p.sum(2)
    tol = ref * (2 * d + (Nq + 128) * 2.0 ** -24) + Nq * 1e-37
    _near(got, ref, tol)
    assert torch.equal(ops.attn_key_weights(q, k, key_bias=bias, causal=causal), got)
    w = _rand((B, H, Nk + 4), 3, 1.0, torch.float32)
    w0 = w.clone()
    assert ops.attn_key_weights(q, k, key_bias=bias, causal=causal, weight=w) is w
    _near(w[..., :Nk], w0[..., :Nk].double() + ref, tol + 2.0 ** -23 * (w0[..., :Nk].double().abs() + ref))
    assert torch.equal(w[..., Nk:], w0[..., Nk:])
    if kind == "all":
        assert bool((got[-1] == 0).all())


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [      # few queries, many keys: row sums by chunks of keys
    (1, 3, 16411, 1, 64, True, "left"), (2, 130, 4100, 2, 128, True, "holes"), (3, 40, 2000, 1, 128, False, "all"), (1, 700, 700, 1, 128, True, None),
    (2, 1, 513, 3, 64, True, "add"), (1, 129, 1025, 40, 128, True, "left")])
def test_attn_key_weights_of_few_queries(B, Nq, Nk, H, hd, causal, kind):
    test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind)


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [      # few keys: one launch; beyond (last two): two
    (2, 1, 33, 3, 128, True, "add"), (3, 31, 97, 2, 64, True, "holes"), (2, 128, 128, 3, 128, True, "left"), (2, 129, 161, 2, 128, True, "all"),
    (1, 256, 256, 2, 64, True, "left"), (2, 200, 256, 2, 128, False, "add"), (2, 353, 384, 3, 128, True, "left"), (1, 384, 384, 2, 64, True, None),
    (1, 800, 65, 3, 128, False, "holes"), (40, 70, 70, 20, 64, True, "add"), (2, 385, 385, 2, 128, True, "left"), (1, 300, 384, 2, 64, False, "add")])
def test_attn_key_weights_of_few_keys(B, Nq, Nk, H, hd, causal, kind):
    test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind)


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [      # more blocks than CUs: one group of waves per workgroup, and (last) two
    (2, 130, 130, 66, 64, True, "left"), (1, 333, 333, 90, 128, True, None), (3, 700, 700, 30, 64, True, "holes"), (2, 200, 650, 130, 64, False, "add"),
    (1, 700, 700, 45, 128, True, "add")])
def test_attn_key_weights_of_many_blocks(B, Nq, Nk, H, hd, causal, kind):
    test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind)


def _ref_evict(w, bias, n, budget, recent):
    """kept rows, by Python sorting"""
    B, H = w.shape[:2]
    w, b = w.cpu(), None if bias is None else bias.cpu()
    kept = torch.empty((B, H, budget), dtype=torch.int32)
    for i in range(B):
        for h in range(H):
            def key(j):
                if b is not None and float(b[i, h, j]) <= -1.0e4:
                    return (2, 0.0, j)
                x = float(w[i, h, j])
                return (1, 0.0, j) if x != x else (0, -x, j)
            first = sorted(range(n - recent), key=key)[:budget - recent]
            kept[i, h] = torch.tensor(sorted(first) + list(range(n - recent, n)), dtype=torch.int32)
    return kept


@pytest.mark.parametrize("B,n,budget,recent,H,hd,masked", [
    (1, 1, 1, 0, 1, 64, False), (1, 2, 1, 0, 2, 128, False), (1, 2, 1, 1, 1, 64, True), (2, 353, 256, 64, 4, 128, False), (3, 100, 100, 0, 2, 64, True),
    (2, 1025, 512, 512, 3, 128, True), (1, 2049, 1, 0, 2, 64, False), (2, 2500, 1111, 7, 2, 128, True), (1, 13000, 900, 100, 1, 64, True),
    (4, 64, 63, 0, 5, 64, False), (1, 512, 300, 9, 2, 128, True), (2, 2048, 2000, 0, 1, 64, True), (1, 4096, 17, 3, 2, 64, True),
    (1, 16384, 16000, 1, 1, 64, False), (2, 17000, 5000, 33, 1, 128, True)])
@pytest.mark.parametrize("inplace", [False, True])
def test_cache_evict_keeps_the_heaviest_rows(B, n, budget, recent, H, hd, masked, inplace):
    rows = n + 6
    k, v = _rand((B, rows, H, hd), 1), _rand((B, rows, H, hd), 2)
    w = _rand((B, H, rows), 3, 1.0, torch.float32)
    w[..., ::3] = 0.0                                                    # ties
    w[..., 1::6] = -0.0
    if n > 50:
        w[..., 7], w[..., 11], w[..., 13] = NAN, INF, -INF
    bias = _bias("left", B * H, rows, 4).view(B, H, rows) if masked else None
    k0, v0, w0, b0 = k.clone(), v.clone(), w.clone(), None if bias is None else bias.clone()
    want = _ref_evict(w[..., :n], None if bias is None else bias[..., :n], n, budget, recent).to(DEV)
    out = None
    if not inplace:
        out = (torch.full((B, budget + 2, H, hd), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((B, budget + 2, H, hd), 7.0, dtype=torch.bfloat16, device=DEV),
               torch.full((B, H, budget + 2), 7.0, device=DEV), torch.full((B, H, budget + 2), 7.0, device=DEV) if masked else None)
    kept = ops.cache_evict(k, v, w, n, budget, recent, key_bias=bias, out=out)
    assert kept.dtype == torch.int32 and torch.equal(kept, want)
    ko, vo, wo, bo = (k, v, w, bias) if inplace else out
    idx = want.long()
    src = idx.transpose(1, 2)[..., None].expand(-1, -1, -1, hd)
    assert torch.equal(ko[:, :budget], k0.gather(1, src)) and torch.equal(vo[:, :budget], v0.gather(1, src))
    assert torch.equal(wo[..., :budget].view(torch.int32), w0.gather(2, idx).view(torch.int32))
    if masked:
        assert torch.equal(bo[..., :budget], b0.gather(2, idx))
    if inplace:
        assert torch.equal(k[:, budget:], k0[:, budget:]) and torch.equal(v[:, budget:], v0[:, budget:])
        assert bool((w[..., budget:n] == 0).all()) and torch.equal(w[..., n:], w0[..., n:])
        assert not masked or (bool((bias[..., budget:n] == 0).all()) and torch.equal(bias[..., n:], b0[..., n:]))
    else:
        assert all(bool((t[:, budget:] == 7.0).all()) for t in out[:2]) and bool((wo[..., budget:] == 7.0).all())
        assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(w.view(torch.int32), w0.view(torch.int32))


@pytest.mark.parametrize("inplace", [False, True])
def test_cache_evict_of_many_long_caches(inplace):
    test_cache_evict_keeps_the_heaviest_rows(1, 16400, 60, 7, 34, 64, True, inplace)


# ---------------------------------------------------------------- the paths that use them: prompts that continue a prefix, bounded caches
def _llm(seed, **kw):
    from dataclasses import replace
    from hawkeye_amd import weights as W
    from hawkeye_amd.config import SMALL_LLM
    from hawkeye_amd.decode import LlamaGenerator
    from hawkeye_amd.llm import LlamaPrefill
    cfg = replace(SMALL_LLM, **kw)
    pre = LlamaPrefill(cfg, DEV).load_state_dict(W.make_llm_state_dict(cfg, seed))
    return cfg, pre, LlamaGenerator(pre)


def _prompt(cfg, P, lengths, seed):
    """One prefix [1, P] with 8 video rows, and questions of the given lengths left-padded to the longest: (prefix, questions, mask, video)"""
    from hawkeye_amd import weights as W
    g = torch.Generator(device="cpu").manual_seed(seed)
    prefix = torch.randint(3, cfg.vocab_size, (1, P), generator=g)
    prefix[0, 5:13] = -torch.arange(1, 9)
    S = max(lengths)
    ask = torch.randint(3, cfg.vocab_size, (len(lengths), S), generator=g)
    mask = (torch.arange(S)[None] >= S - torch.tensor(lengths)[:, None]).long()
    ask[mask == 0] = 2
    return prefix.to(DEV), ask.to(DEV), mask.to(DEV), W._normal("video_tokens", seed, (8, cfg.hidden_size), 0.05).to(DEV)


def _rel(a, ref):
    return ((a.double() - ref.double()).abs().max() / ref.double().abs().max()).item()


@pytest.mark.parametrize("P,lengths", [(60, [17, 17, 17]), (100, [40]), (33, [5, 20, 1, 12]), (90, [70] * 3), (64, [3] * 16)])
def test_prompts_that_continue_a_prefix_equal_whole_prompts(P, lengths):
    """make_prefix + prefill / generate(prefix=): logits, hidden states and tokens of the same prompts written out in full."""
    cfg, pre, gen = _llm(21)
    prefix, ask, mask, video = _prompt(cfg, P, lengths, 21)
    B, S, T = len(lengths), max(lengths), 6
    ragged = min(lengths) < S
    whole = torch.cat([prefix.expand(B, P), ask], 1)
    wmask = None
    if ragged:                                                # whole prompts left-pad in front of the prefix
        for b, n in enumerate(lengths):
            whole[b] = torch.cat([torch.full((S - n,), 2, device=DEV), prefix[0], ask[b, S - n:]])
        wmask = torch.cat([torch.ones_like(whole[:, :P]), torch.ones_like(mask)], 1)
        for b, n in enumerate(lengths):
            wmask[b, :S - n] = 0
    ref = gen.generate(src=whole, video=video, attention_mask=wmask, max_new_tokens=T, return_logits=True)
    full = pre.prefill(src=whole, video=video, attention_mask=wmask, position_ids="generate" if ragged else None)
    hidden = full["hidden"][:, P:].clone()
    pf = pre.make_prefix(src=prefix, video=video)
    assert pf.rows == pf.n_positions == P and pf.kept is None
    out = pre.prefill(src=ask, attention_mask=mask if ragged else None, position_ids="generate" if ragged else None, prefix=pf)
    # two kernels for one operator: bf16 products and residual stream differ by their roundings (the tolerance of the cache tests)
    valid = mask.bool()
    assert _rel(out["hidden"][valid], hidden[valid]) < 2e-2 and _rel(out["logits"], ref["logits"][0]) < 2e-2
    got = gen.generate(src=ask, attention_mask=mask if ragged else None, prefix=pf, max_new_tokens=T, forced_tokens=ref["tokens"], return_logits=True)
    for t in range(T):
        assert _rel(got["logits"][t], ref["logits"][t]) < 2e-2, t
    again = gen.generate(src=ask, attention_mask=mask if ragged else None, prefix=pf, max_new_tokens=T, forced_tokens=ref["tokens"], return_logits=True)
    assert torch.equal(again["logits"], got["logits"])
    free = gen.generate(src=ask, attention_mask=mask if ragged else None, prefix=pf, max_new_tokens=T)["tokens"]
    top2 = ref["logits"].topk(2, -1).values
    sure = ((top2[..., 0] - top2[..., 1]) / ref["logits"].abs().amax(-1) > 5e-2).t()      # [B, T]
    for b in range(B):
        for t in range(T):
            if not bool(sure[b, t]):
                break                                         # what follows depends on a near-tie
            assert free[b, t] == ref["tokens"][b, t], (b, t)


def test_a_prefix_cut_to_its_own_length_less_nothing_is_the_prefix():
    cfg, pre, gen = _llm(22)
    prefix, ask, mask, video = _prompt(cfg, 70, [12, 12], 22)
    a, b = pre.make_prefix(src=prefix, video=video), pre.make_prefix(src=prefix, video=video, budget=70)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    cut = pre.make_prefix(src=prefix, video=video, budget=40, recent=10)
    assert cut.rows == 40 and cut.n_positions == 70 and tuple(cut.kept.shape) == (cfg.num_hidden_layers, cfg.num_attention_heads, 40)
    hd = cfg.head_dim
    for layer in range(cfg.num_hidden_layers):
        for h in range(cfg.num_attention_heads):
            rows = cut.kept[layer, h].long()
            assert torch.equal(cut.k[layer, :, h * hd:(h + 1) * hd], a.k[layer, rows, h * hd:(h + 1) * hd])
            assert torch.equal(cut.v[layer, :, h * hd:(h + 1) * hd], a.v[layer, rows, h * hd:(h + 1) * hd])
            assert rows[-10:].tolist() == list(range(60, 70)) and bool((rows[1:] > rows[:-1]).all())
    # the kept rows are those the prompt's own queries weigh most
    pre.prefill(src=prefix, video=video)
    qkv = pre.last_ws["qkv"].view(cfg.num_hidden_layers, 70, 3, cfg.num_attention_heads, hd)
    p, _ = _ref_weights(qkv[:, :, 0], qkv[:, :, 1], None, True)
    w = p.sum(2)
    inside = torch.zeros_like(w, dtype=torch.bool).scatter_(2, cut.kept.long(), True)
    for layer in range(cfg.num_hidden_layers):
        for h in range(cfg.num_attention_heads):
            old = torch.arange(70, device=DEV) < 60
            assert float(w[layer, h][inside[layer, h] & old].min()) >= float(w[layer, h][~inside[layer, h] & old].max()) * (1 - 1e-4)
    out = gen.generate(src=ask, prefix=cut, max_new_tokens=3, return_logits=True)
    assert bool(torch.isfinite(out["logits"]).all()) and out["tokens"].shape == (2, 3)
    with pytest.raises(RuntimeError, match="budget=0"):
        pre.make_prefix(src=prefix, video=video, budget=0)
    with pytest.raises(RuntimeError, match="window=0"):
        pre.make_prefix(src=prefix, video=video, budget=5, window=0)
    with pytest.raises(RuntimeError, match="together"):
        gen.generate(src=ask, prefix=cut, cache_budget=20, max_new_tokens=2)
    with pytest.raises(RuntimeError, match="exceeds max_position_embeddings"):
        gen.generate(src=ask, prefix=cut, max_new_tokens=200)
    with pytest.raises(RuntimeError, match="left-padded"):
        m = mask.clone()
        m[0, 0] = 0
        pre.prefill(src=ask, attention_mask=m, prefix=cut)


@pytest.mark.parametrize("masked", [False, True])
def test_a_budget_that_never_binds_changes_nothing(masked):
    cfg, pre, gen = _llm(23)
    prefix, ask, mask, video = _prompt(cfg, 40, [50, 50] if not masked else [50, 31, 8], 23)
    kw = dict(src=ask, attention_mask=mask if masked else None, max_new_tokens=8, return_logits=True)
    ref = gen.generate(**kw)
    got = gen.generate(cache_budget=100, forced_tokens=ref["tokens"], **kw)
    for t in range(8):
        assert _rel(got["logits"][t], ref["logits"][t]) < 2e-2, t


@pytest.mark.parametrize("lengths", [[90], [60, 60, 60], [70, 22, 41]])
def test_a_bounded_cache_follows_its_definition_step_by_step(lengths):
    """generate(cache_budget=): the caches after every cut, against a 64-bit bookkeeping of weights over the same keys."""
    budget, recent, T = 24, 8, 150
    cfg, pre, gen = _llm(24)
    _, ask, mask, video = _prompt(cfg, 20, lengths, 24)
    masked = min(lengths) < max(lengths)
    B, S, Lyr, H, hd = len(lengths), max(lengths), cfg.num_hidden_layers, cfg.num_attention_heads, cfg.head_dim
    kw = dict(src=ask, attention_mask=mask if masked else None, cache_budget=budget, cache_recent=recent)
    cuts = []
    whole = ops.cache_evict

    def spy(k, v, w, n, b, r=0, key_bias=None, out=None):
        before = (k[:, :n].clone(), v[:, :n].clone(), w[..., :n].clone(), None if key_bias is None else key_bias[..., :n].clone())
        kept = whole(k, v, w, n, b, r, key_bias=key_bias, out=out)
        ko, vo = (k, v) if out is None else out[:2]
        cuts.append((before, n, kept.clone(), ko[:, :b].clone(), vo[:, :b].clone()))
        return kept

    ops.cache_evict = spy
    try:
        out = gen.generate(max_new_tokens=T, return_logits=True, **kw)
    finally:
        ops.cache_evict = whole
    assert out["tokens"].shape == (B, T) and bool(torch.isfinite(out["logits"]).all())
    assert len(cuts) == 1 + (T - 2) // 64                      # the prompt's, then every 64 steps
    for (k0, v0, w0, b0), n, kept, ko, vo in cuts:
        want = _ref_evict(w0, b0, n, budget, recent).to(DEV)
        assert torch.equal(kept, want)
        src = want.long().transpose(1, 2)[..., None].expand(-1, -1, -1, hd)
        assert torch.equal(ko, k0.gather(1, src)) and torch.equal(vo, v0.gather(1, src))
    # the weights themselves: before the first cut in place they are the kept prompt weights plus 64 steps', whose sum over the live
    # keys is one per step (and the prompt's queries gave one each in all)
    first, second = cuts[0], cuts[1]
    kept_w = first[0][2].double().gather(2, first[2].long())
    grown = second[0][2].double().sum(-1) - kept_w.sum(-1)
    assert float((grown - 64).abs().max()) < 64 * (budget + 64 + 128) * 2.0 ** -24 + float(kept_w.sum(-1).max()) * 2.0 ** -18
    valid = torch.tensor(lengths, dtype=torch.float64, device=DEV).repeat(Lyr)[:, None]
    tot = first[0][2].double()
    if masked:                                                 # a padded query sees removed keys only and adds nothing
        assert float((tot.masked_select(first[0][3] <= -1.0e4)).abs().max()) == 0.0
    assert float((tot.sum(-1) - valid).abs().max()) < S * 2.0 ** -12
    # what was not cut yet equals the unbounded run: token 0 comes from the same prefill
    ref = gen.generate(src=ask, attention_mask=mask if masked else None, max_new_tokens=1, return_logits=True)
    assert torch.equal(ref["logits"][0], out["logits"][0])
    with pytest.raises(RuntimeError, match="cache_budget=0"):
        gen.generate(src=ask, cache_budget=0, max_new_tokens=2)
    with pytest.raises(RuntimeError, match="needs cache_budget"):
        gen.generate(src=ask, cache_recent=3, max_new_tokens=2)


def test_plans_of_many_prefixes_stay_bounded():
    from hawkeye_amd.llm import MAX_PLANS
    cfg, pre, gen = _llm(25)
    prefix, ask, _, video = _prompt(cfg, 100, [4, 4], 25)
    first = None
    for P in list(range(20, 20 + MAX_PLANS + 3)) + [20]:
        pf = pre.make_prefix(src=prefix[:, :P], video=video)
        out = gen.generate(src=ask, prefix=pf, max_new_tokens=2, return_logits=True)
        if P == 20 and first is None:
            first = out
    assert len(gen.plans) <= MAX_PLANS and len(pre.plans) <= MAX_PLANS
    assert torch.equal(out["logits"], first["logits"]) and torch.equal(out["tokens"], first["tokens"])


def test_streams_graphs_and_strides():
    """Another stream, a captured call replayed with eager work between, and caches whose offsets pass 2^31 elements."""
    B, H, hd, P, n = 3, 2, 128, 300, 90
    q, kp, vp = _rand((B, 1, H, hd), 1, 0.2), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    k, v = _rand((B, n, H, hd), 4), _rand((B, n, H, hd), 5)
    w = _rand((B, H, n), 6, 1.0, torch.float32).abs()

    def run(wo, kc, vc, ww):
        a = ops.prefix_attention(q, kp, vp, k, v)
        wk = ops.attn_key_weights(q, k)
        o = ops.decode_attn_weights(q.view(B, H * hd), k.view(B, n, H * hd), v.view(B, n, H * hd), n, H, hd, w, weight_out=wo)
        kept = ops.cache_evict(k, v, wo, n, 40, 9, out=(kc, vc, ww, None))
        return a, wk, o, kept

    def bufs():
        return torch.empty_like(w), torch.empty((B, 40, H, hd), dtype=torch.bfloat16, device=DEV), torch.empty((B, 40, H, hd), dtype=torch.bfloat16, device=DEV), \
            torch.empty((B, H, 40), device=DEV)
    base_b = bufs()
    base = [t.clone() for t in run(*base_b)] + [t.clone() for t in base_b]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other_b = bufs()
    with torch.cuda.stream(side):
        other = run(*other_b)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, list(other) + list(other_b)))
    graph_b = bufs()
    with torch.cuda.stream(side):
        run(*graph_b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = run(*graph_b)
    q0 = q.clone()
    for rep in range(4):
        q.copy_(q0 * (1 + rep))
        want = [t.clone() for t in run(*base_b)] + [t.clone() for t in base_b]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, list(res) + list(graph_b))), rep
    # a cache of 2^31 elements and more per tensor: the rows used lie behind the 32-bit offsets
    H, hd, rows = 32, 128, 300000
    big = torch.zeros((2, rows, H * hd), dtype=torch.bfloat16, device=DEV)              # 2.46e9 elements, sequence 1 behind 1.2e9
    bigv = torch.zeros_like(big)
    n = 70
    kk, vv = _rand((2, n, H * hd), 7), _rand((2, n, H * hd), 8)
    big[:, rows - n:], bigv[:, rows - n:] = kk, vv
    qq = _rand((2, 1, H, hd), 9, 0.2)
    got = ops.prefix_attention(qq, kp[:0].new_empty((0, H, hd)), vp[:0].new_empty((0, H, hd)), big[:, rows - n:].unflatten(2, (H, hd)), bigv[:, rows - n:].unflatten(2, (H, hd)))
    assert torch.equal(got, ops.prefix_attention(qq, kp[:0].new_empty((0, H, hd)), vp[:0].new_empty((0, H, hd)), kk.unflatten(2, (H, hd)), vv.unflatten(2, (H, hd))))
    flat = big.view(-1, H, hd)                                                          # one prefix of 600000 rows, its end used
    got = ops.prefix_attention(qq, flat[-n:], bigv.view(-1, H, hd)[-n:], kk.unflatten(2, (H, hd)), vv.unflatten(2, (H, hd)))
    assert torch.equal(got, ops.prefix_attention(qq, kk[1].unflatten(1, (H, hd)), vv[1].unflatten(1, (H, hd)), kk.unflatten(2, (H, hd)), vv.unflatten(2, (H, hd))))
    wbig = torch.zeros((2, H, rows), device=DEV)
    o = ops.decode_attn_weights(qq.view(2, -1), big, bigv, rows, H, hd, wbig, key_bias=torch.cat([torch.full((2, rows - n), -1.0e4, device=DEV), torch.zeros((2, n), device=DEV)], 1))
    ref, tol = _ref_prefix(qq, kp[:0].new_empty((0, H, hd)), vp[:0].new_empty((0, H, hd)), kk.unflatten(2, (H, hd)), vv.unflatten(2, (H, hd)), None)
    _near(o.view(2, 1, H, hd), ref, tol)
    assert float((wbig.sum(-1) - 1).abs().max()) < 1e-4 and bool((wbig[..., :rows - n] == 0).all())
    kept = ops.cache_evict(big.unflatten(2, (H, hd)), bigv.unflatten(2, (H, hd)), wbig, rows, 50, 20)
    assert bool((kept[..., -20:] == torch.arange(rows - 20, rows, device=DEV)).all()) and bool((kept >= rows - n).all())
    src = (kept.long() - (rows - n)).transpose(1, 2)[..., None].expand(-1, -1, -1, hd)
    assert torch.equal(big[:, :50].unflatten(2, (H, hd)), kk.unflatten(2, (H, hd)).gather(1, src))


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [      # keys too many for one launch, too few for chunks, few rows: the smallest workspaces
    (1, 1, 400, 4, 64, True, None), (2, 1, 400, 2, 128, True, "left"), (1, 4, 385, 1, 128, True, None), (4, 1, 430, 1, 64, False, "holes"), (1, 1, 448, 4, 128, True, "add")])
def test_attn_key_weights_with_the_smallest_workspaces(B, Nq, Nk, H, hd, causal, kind):
    test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind)


def test_outputs_in_other_orders_of_their_dims():
    """Tokens outside sequences, heads outside sequences: the results of the plain layouts."""
    B, Nq, P, Nk, H, hd = 3, 5, 600, 40, 4, 64
    q, kp, vp = _rand((B, Nq, H, hd), 1, 0.2), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    k, v = _rand((B, Nk, H, hd), 4), _rand((B, Nk, H, hd), 5)
    out = torch.full((Nq, B, H, hd), 7.0, dtype=torch.bfloat16, device=DEV)
    want = ops.prefix_attention(q, kp, vp, k, v)
    assert torch.equal(ops.prefix_attention(q, kp, vp, k, v, out=out.transpose(0, 1)), want)
    w = ops.attn_key_weights(q, k)
    wt = torch.zeros((H, B, Nk), device=DEV)
    assert torch.equal(ops.attn_key_weights(q, k, weight_out=wt.transpose(0, 1)), w)
    kc, vc, q1 = k.reshape(B, Nk, H * hd), v.reshape(B, Nk, H * hd), q[:, 0].reshape(B, H * hd).contiguous()
    w2 = w.clone()
    o = ops.decode_attn_weights(q1, kc, vc, Nk, H, hd, w2)
    assert torch.equal(ops.decode_attn_weights(q1, kc, vc, Nk, H, hd, wt.transpose(0, 1)), o) and torch.equal(wt.transpose(0, 1), w2)
    ko, vo = torch.empty((11, B, H, hd), dtype=torch.bfloat16, device=DEV), torch.empty((11, B, H, hd), dtype=torch.bfloat16, device=DEV)
    wo = torch.empty((H, B, 11), device=DEV)
    kept = ops.cache_evict(k, v, wt.transpose(0, 1), Nk, 11, 3, out=(ko.transpose(0, 1), vo.transpose(0, 1), wo.transpose(0, 1), None))
    assert torch.equal(ops.cache_evict(k, v, w2, Nk, 11, 3), kept)            # in place
    assert torch.equal(ko.transpose(0, 1), k[:, :11]) and torch.equal(vo.transpose(0, 1), v[:, :11]) and torch.equal(wo.transpose(0, 1), w2[..., :11])


def _deep(B, n, first, seed):
    """Biases of about -9000 (far below all scores, and still there) on the first `first` keys, 0 on the others."""
    b = torch.zeros((B, n), device=DEV)
    b[:, :first] = -9000.0 + _rand((B, first), seed, 2.0, torch.float32)
    return b


# Two sizes of reference points in one row.  A row that sees an ordinary key has nothing left of the others: the tolerance is the usual one.  (Few
# ordinary keys and queries: errors of many would cancel.)
@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,first", [
    (2, 3, 460, 4, 128, True, 448), (3, 2, 700, 5, 64, False, 690), (2, 7, 500, 3, 128, False, 450), (70, 2, 450, 5, 64, True, 440), (2, 5, 5000, 2, 128, True, 4990),
    (40, 3, 700, 64, 128, False, 699), (2, 500, 700, 70, 64, True, 150), (2, 100, 300, 2, 128, True, 100), (1, 20, 100, 2, 64, False, 70)])
def test_attn_key_weights_behind_keys_with_large_biases(B, Nq, Nk, H, hd, causal, first):
    q, k = _rand((B, Nq, H, hd), 1, 0.05 * hd ** -0.5), _rand((B, Nk, H, hd), 2)
    # (small scores: a small d)
    bias = _deep(B, Nk, first, 3)
    got = ops.attn_key_weights(q, k, key_bias=bias, causal=causal)
    p, d = _ref_weights(q, k, bias, causal)
    ref = p.sum(2)
    _near(got, ref, ref * (2 * d + (Nq + 128) * 2.0 ** -24) + Nq * 1e-37)


# A row that sees biased keys alone: its scores lie below 2^14 and are held in 32 bits with the bias in them, 2^-11 for each of five roundings (the
# product with log2 e, the addition, in both passes; the row's sum).
@pytest.mark.parametrize("B,Nq,Nk,H,hd,first", [(2, 500, 500, 2, 128, 300), (1, 130, 600, 2, 64, 600), (2, 100, 100, 3, 128, 50), (1, 30, 3000, 1, 64, 3000)])
def test_attn_key_weights_of_rows_with_large_biases_alone(B, Nq, Nk, H, hd, first):
    q, k = _rand((B, Nq, H, hd), 1, 1.5 * hd ** -0.5 * LOG2E), _rand((B, Nk, H, hd), 2)
    bias = _deep(B, Nk, first, 3)
    got = ops.attn_key_weights(q, k, key_bias=bias)
    p, d = _ref_weights(q, k, bias, True)
    ref = p.sum(2)
    _near(got, ref, ref * (2 * d + (Nq + 128) * 2.0 ** -24 + 5 * math.log(2.0) * 2.0 ** -11) + Nq * 1e-37)



# Questions whose own keys all carry large biases, or begin with them: what the biases have in common drops out of a softmax, and takes no bit along.
@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,first,rest", [
    (2, 70, 0, 200, 3, 128, 1e5, 1e5), (3, 130, 300, 130, 4, 64, 1e5, 1e5), (2, 40, 0, 400, 90, 128, 1e5, 1e5), (1, 257, 0, 460, 8, 64, 3e4, 1e5), (2, 100, 64, 300, 2, 128, -9000.0, 0.0),
    (1, 64, 0, 3000, 1, 64, 1e5, 1e5)])
def test_prefix_attention_of_questions_with_large_biases(B, Nq, P, Nk, H, hd, first, rest):
    q, kp, vp = _rand((B, Nq, H, hd), 1, 1.5 * hd ** -0.5 * LOG2E), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    k, v = _rand((B, Nk, H, hd), 4), _rand((B, Nk, H, hd), 5)
    bias = torch.full((B, Nk), float(rest), device=DEV)
    bias[:, :Nk - Nq - 1] = float(first)
    bias += _rand((B, Nk), 6, 2.0, torch.float32)
    v[..., ::2] = 3.0 * torch.sign(q[:1, :1, :, ::2]) + v[..., ::2]           # (outputs far from zero)
    got = ops.prefix_attention(q, kp, vp, k, v, key_bias=bias)
    ref, tol = _ref_prefix(q, kp, vp, k, v, bias)
    _near(got, ref, tol)


# Steps and a few tokens: P is two bf16 numbers, off by 2^-16 of itself.  What is left beside the output's own rounding: scores (d), sums of n terms in
# 32 bits in numerator and denominator, exp2 of the terms, chunks and waves (2^-20 covers eight of them).
def _near_32(got, ref, A, d, n):
    _near(got, ref, 2.0 ** -8 * ref.abs() + 1.01 * A * (2.0 ** -16 + 2 * d + 2 * (n + 64) * 2.0 ** -24 + 2.0 ** -20) + 1e-37)


@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", [
    (4, 1, 352, 20, 32, 128, None), (16, 1, 1985, 61, 8, 128, "left"), (16, 1, 1985, 61, 8, 128, None), (5, 3, 777, 130, 12, 64, "add"), (1, 1, 5000, 300, 4, 128, "holes"),
    (4, 16, 1500, 16, 4, 64, None), (3, 1, 0, 90, 4, 128, "left"), (40, 1, 100, 33, 3, 128, "left"), (2, 32, 300, 32, 3, 64, None)])
def test_steps_keep_the_bits_of_their_probabilities(B, Nq, P, Nk, H, hd, kind):
    q, kp, vp = _rand((B, Nq, H, hd), 1, 0.2 * hd ** -0.5 * LOG2E), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
    k, v, bias = _rand((B, Nk, H, hd), 4), _rand((B, Nk, H, hd), 5), _bias(kind, B, Nk, 6)
    got = ops.prefix_attention(q, kp, vp, k, v, key_bias=bias)
    p = _softmax(_h(q), [_h(kp[None]).expand(B, -1, -1, -1), _h(k)], [None, None if bias is None else bias.double()[:, None, None]], Nq)
    vs = torch.cat([_h(vp[None]).expand(B, -1, -1, -1), _h(v)], 2)
    d = _d(_h(q), [_h(kp[None]).expand(B, -1, -1, -1), _h(k)], hd)
    _near_32(got.transpose(1, 2), p @ vs, p @ vs.abs(), d, P + Nk)


@pytest.mark.parametrize("B,n,H,hd,kind", [(1, 353, 8, 128, None), (4, 1500, 4, 128, "left"), (2, 1500, 4, 128, None), (3, 700, 5, 64, "add"), (1, 9000, 2, 64, None)])
def test_weighted_steps_keep_the_bits_of_their_probabilities(B, n, H, hd, kind):
    q = _rand((B, H * hd), 1, 0.2 * hd ** -0.5 * LOG2E)
    k, v, bias = _rand((B, n, H * hd), 2), _rand((B, n, H * hd), 3), _bias(kind, B, n, 4)
    out = ops.decode_attn_weights(q, k, v, n, H, hd, torch.zeros((B, H, n), device=DEV), key_bias=bias)
    p, d = _ref_weights(q.view(B, 1, H, hd), k.view(B, n, H, hd), bias, False)
    vd = _h(v.view(B, n, H, hd))
    _near_32(out.view(B, H, hd), (p @ vd)[:, :, 0], (p @ vd.abs())[:, :, 0], d, n)


@pytest.mark.parametrize("form", ["rows", "blocks", "qkv"])
@pytest.mark.parametrize("B,n,budget,H,hd", [(2, 300, 100, 3, 64), (3, 700, 513, 2, 128), (12, 1500, 900, 3, 128), (1, 17000, 300, 2, 64)])
def test_cache_evict_of_interleaved_caches(form, B, n, budget, H, hd):
    """K and V as views of one tensor, in place and into views of one tensor: the results of two tensors."""
    rows = n + 2
    kv = _rand((B, 2, rows, H, hd) if form == "blocks" else (B, rows, 2 if form == "rows" else 3, H, hd), 1)
    k, v = (kv[:, 0], kv[:, 1]) if form == "blocks" else (kv[:, :, -2], kv[:, :, -1])
    w = _rand((B, H, rows), 3, 1.0, torch.float32).abs()
    k1, v1, w1, kv0 = k.clone(), v.clone(), w.clone(), kv.clone()
    want = ops.cache_evict(k1, v1, w1, n, budget, 20)
    new = torch.full((B, 2, budget + 1, H, hd) if form == "blocks" else (B, budget + 1, 2, H, hd), 7.0, dtype=torch.bfloat16, device=DEV)
    ko, vo = (new[:, 0], new[:, 1]) if form == "blocks" else (new[:, :, 0], new[:, :, 1])
    wo = torch.empty((B, H, budget), device=DEV)
    assert torch.equal(ops.cache_evict(k, v, w, n, budget, 20, out=(ko, vo, wo, None)), want)
    assert torch.equal(kv, kv0)
    for a, b, c in ((ko, k1, vo), (vo, v1, ko)):
        assert torch.equal(a[:, :budget], b[:, :budget]) and bool((a[:, budget:] == 7.0).all())
    assert torch.equal(wo, w1[..., :budget])
    assert torch.equal(ops.cache_evict(k, v, w, n, budget, 20), want)
    assert torch.equal(k, k1) and torch.equal(v, v1) and torch.equal(w, w1)
    if form == "qkv":
        assert torch.equal(kv[:, :, 0], kv0[:, :, 0])


def test_prefix_attention_into_a_column_of_its_inputs_tensor():
    B, n, H, hd = 3, 40, 2, 128
    x = _rand((B, n, 4, H, hd), 1, 0.3)
    kp, vp = _rand((500, H, hd), 2), _rand((500, H, hd), 3)
    x0 = x.clone()
    want = ops.prefix_attention(x0[:, :, 0], kp, vp, x0[:, :, 1], x0[:, :, 2])
    got = ops.prefix_attention(x[:, :, 0], kp, vp, x[:, :, 1], x[:, :, 2], out=x[:, :, 3])
    assert torch.equal(got, want) and torch.equal(x[:, :, :3], x0[:, :, :3])
    with pytest.raises(RuntimeError, match="overlaps an input"):
        ops.prefix_attention(x[:, :, 0], kp, vp, x[:, :, 1], x[:, :, 2], out=x[:, :, 2])


# What the cases above leave out of the rules that pick a kernel.  Questions of a usual prompt without padding (two groups of waves, and one), heads
# of 64 with biases in two groups; rows of more than 16 sequences' tokens over row blocks with the own keys by workgroup; steps over a long prefix with
# heads of 64; many sequences without a prefix.
@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", [
    (1, 37, 352, 37, 32, 128, None), (4, 64, 352, 64, 8, 128, None), (8, 128, 352, 128, 32, 128, None), (1, 64, 352, 64, 16, 64, "add"), (3, 130, 352, 130, 8, 64, "left"), (2, 257, 64, 257, 3, 64, "left"),
    (8, 130, 200, 130, 2, 64, "add"), (3, 33, 200, 33, 3, 128, None), (2, 257, 0, 257, 70, 128, None), (1, 100, 0, 500, 4, 64, "all"), (2, 200, 2000, 200, 2, 64, None), (32, 16, 1600, 40, 4, 128, None), (32, 16, 1600, 40, 4, 128, "left"), (16, 32, 1600, 40, 6, 128, None),
    (16, 32, 1600, 40, 6, 128, "holes"), (32, 16, 2100, 130, 8, 64, None), (32, 16, 2100, 130, 8, 64, "add"), (16, 25, 3000, 200, 8, 64, None), (16, 25, 3000, 200, 8, 64, "all"),
    (40, 16, 1300, 30, 26, 64, None), (40, 16, 1300, 30, 26, 64, "left"), (40, 16, 600, 30, 26, 128, None), (33, 17, 800, 17, 20, 128, None), (5, 3, 1500, 40, 6, 64, None),
    (5, 3, 1500, 40, 6, 64, "left"), (40, 1, 0, 40, 30, 128, "all"), (40, 1, 0, 90, 30, 128, None), (60, 3, 0, 33, 20, 64, "left"), (60, 1, 0, 33, 20, 64, None),
    (40, 5, 0, 500, 20, 64, "holes"), (3, 1, 1500, 40, 8, 128, None)])
def test_prefix_attention_by_every_rule(B, Nq, P, Nk, H, hd, kind):
    test_prefix_attention_matches_its_definition(B, Nq, P, Nk, H, hd, kind)


@pytest.mark.parametrize("B,Nq,Nk,H,hd,causal,kind", [      # without biases: two launches of one group and of two, chunks, one launch of up to 256 keys
    (2, 450, 450, 45, 128, True, None), (2, 450, 450, 45, 64, True, None), (1, 1000, 1000, 2, 64, True, None), (2, 40, 3000, 2, 64, True, None), (1, 600, 600, 4, 64, False, None),
    (2, 200, 250, 2, 128, True, None), (1, 256, 256, 3, 64, True, None), (64, 400, 400, 8, 128, True, None)])
def test_attn_key_weights_without_biases(B, Nq, Nk, H, hd, causal, kind):
    test_attn_key_weights_matches_its_definition(B, Nq, Nk, H, hd, causal, kind)


@pytest.mark.parametrize("B,n,budget,recent,H,hd,masked", [      # many rows per workgroup: several ordered steps, where more than 32 pairs move them in place
    (2, 576, 512, 128, 20, 128, True), (2, 576, 512, 128, 20, 128, False), (1, 2048, 1900, 5, 34, 64, True), (2, 600, 200, 9, 2, 128, True), (2, 1000, 500, 3, 3, 64, False), (2, 512, 400, 3, 3, 64, True),
    (2, 2500, 1500, 7, 20, 128, True), (2, 2500, 200, 7, 2, 128, False), (1, 3000, 2500, 0, 3, 64, False), (1, 5000, 3000, 7, 34, 64, False), (1, 6000, 4500, 100, 33, 128, True),
    (1, 13000, 200, 9, 2, 128, True), (1, 9000, 4000, 0, 3, 128, False)])
@pytest.mark.parametrize("inplace", [False, True])
def test_cache_evict_of_many_rows(B, n, budget, recent, H, hd, masked, inplace):
    test_cache_evict_keeps_the_heaviest_rows(B, n, budget, recent, H, hd, masked, inplace)


@pytest.mark.parametrize("B,n,budget,recent,H,hd,masked,inplace", [(1, 16500, 3000, 7, 34, 64, False, True), (1, 16400, 2100, 0, 33, 128, True, True)])
def test_cache_evict_of_many_rows_of_many_long_caches(B, n, budget, recent, H, hd, masked, inplace):
    test_cache_evict_keeps_the_heaviest_rows(B, n, budget, recent, H, hd, masked, inplace)


def test_prefix_attention_in_a_workspace_of_the_callers():
    """Of exactly the size asked for, between guards; too small, of another type, strided: refused."""
    for B, Nq, P, Nk, H, hd in ((16, 1, 1985, 61, 4, 128), (7, 37, 1201, 37, 8, 128), (32, 16, 1600, 40, 4, 128), (5, 3, 1500, 40, 6, 64)):
        need = ops.prefix_attention_ws(B, H, Nq, P, Nk, hd)
        assert need > 64
        q, kp, vp = _rand((B, Nq, H, hd), 1, 0.1), _rand((P, H, hd), 2), _rand((P, H, hd), 3)
        k, v = _rand((B, Nk, H, hd), 4), _rand((B, Nk, H, hd), 5)
        buf = torch.full((need + 512,), 255, dtype=torch.uint8, device=DEV)                   # (as floats: NaN)
        want = ops.prefix_attention(q, kp, vp, k, v)
        for _ in range(2):
            assert torch.equal(ops.prefix_attention(q, kp, vp, k, v, ws=buf[256:256 + need]), want)
            assert bool((buf[:256] == 255).all()) and bool((buf[256 + need:] == 255).all())
        with pytest.raises(RuntimeError, match="workspace"):
            ops.prefix_attention(q, kp, vp, k, v, ws=buf[256:256 + need - 1])
        with pytest.raises(RuntimeError, match="uint8"):
            ops.prefix_attention(q, kp, vp, k, v, ws=torch.empty((need,), device=DEV))
        with pytest.raises(RuntimeError, match="uint8"):
            ops.prefix_attention(q, kp, vp, k, v, ws=torch.empty((2 * need,), dtype=torch.uint8, device=DEV)[::2])
    q = _rand((4, 1, 4, 128), 1, 0.1)
    kp, k = _rand((300, 4, 128), 2), _rand((4, 20, 4, 128), 4)                                # one launch: whatever is passed is left alone
    buf = torch.full((64,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(ops.prefix_attention(q, kp, kp, k, k, ws=buf), ops.prefix_attention(q, kp, kp, k, k)) and bool((buf == 255).all())


@pytest.mark.parametrize("B,Nq,P,Nk,H,hd,kind", [           # the prefix by blocks of 128 rows
    (64, 1, 5000, 40, 16, 128, None), (64, 1, 5000, 140, 16, 128, "left"), (130, 1, 2600, 20, 32, 64, None), (130, 1, 2600, 20, 32, 64, "add"), (256, 1, 200, 30, 64, 128, None)])
def test_steps_of_many_sequences_keep_the_bits_of_their_probabilities(B, Nq, P, Nk, H, hd, kind):
    test_steps_keep_the_bits_of_their_probabilities(B, Nq, P, Nk, H, hd, kind)
