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
