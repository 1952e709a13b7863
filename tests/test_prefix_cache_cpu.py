"""Refusals of the shared-prefix attention, key-weight and eviction entry points: all on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from hawkeye_amd import lib as L
from hawkeye_amd import ops

A = 1 << 20        # stands for an aligned device address: no refused call looks at it


def _refused(rc, text):
    assert rc == 1 and text in L.last_error(), (rc, L.last_error())


def _prefix(**kw):
    H, hd, B, Nq, P, Nk = (kw.get(k, d) for k, d in (("H", 2), ("head_dim", 64), ("B", 2), ("Nq", 1), ("P", 1000), ("Nk", 4)))      # (keys in chunks: a call with a workspace)
    row = H * hd
    base = dict(Q=A, KP=2 * A, VP=3 * A, K=4 * A, V=5 * A, O=6 * A, key_bias=None, ws=8 * A, ws_bytes=1 << 30, B=B, H=H, Nq=Nq, P=P, Nk=Nk,
                head_dim=hd, ldq=row, bsq=row * Nq, ldkp=row, ldvp=row, ldk=row, bsk=row * Nk, ldv=row, bsv=row * Nk, ldo=row, bso=row * Nq,
                bias_bs=Nk)
    base.update(kw)
    return L.load().hk_prefix_attn_bf16(C.byref(L.HkPrefixAttnDesc(**base)), None)


@pytest.mark.parametrize("kw,text", [
    (dict(Q=None), "null operand"), (dict(KP=None), "null prefix"), (dict(head_dim=96), "bad shape"), (dict(Nk=0, Nq=1), "bad shape"), (dict(P=-1), "bad shape"),
    (dict(B=0), "bad shape"), (dict(B=1 << 15, H=1 << 13, Nq=1), "bad shape"), (dict(ldk=129), "strides"), (dict(bsv=-64), "strides"), (dict(bso=64), "rows must not overlap"),
    (dict(ldkp=1 << 25), "2^25"), (dict(Q=A + 8), "aligned"), (dict(ws=8 * A + 8), "aligned"), (dict(ws=None), "workspace"), (dict(ws_bytes=64), "workspace"),
    (dict(O=4 * A), "overlaps an input"), (dict(O=A), "overlaps an input"), (dict(ws=2 * A), "overlaps an input"), (dict(O=8 * A), "output overlaps the workspace")])
def test_prefix_attention_refuses(kw, text):
    _refused(_prefix(**kw), text)
    assert L.load().hk_prefix_attn_bf16(None, None) == 1


def test_workspace_queries_refuse_with_zero():
    lib = L.load()
    assert lib.hk_prefix_attn_ws(2, 2, 1, 8, 4, 64) > 0 and lib.hk_decode_attn_weights_ws(2, 2, 128, 5) > 0
    assert lib.hk_prefix_attn_ws(2, 2, 5, 8, 4, 64) == 0 and lib.hk_prefix_attn_ws(2, 2, 1, 8, 4, 80) == 0 and lib.hk_decode_attn_weights_ws(1, 1, 64, 0) == 0
    assert lib.hk_attn_key_weights_ws(1, 1, 0, 4, 0) == 0 == lib.hk_attn_key_weights_ws(1, 1, 5, 4, 1) and lib.hk_attn_key_weights_ws(2, 3, 5, 7, 1) == L.HK_NO_WS
    assert lib.hk_attn_key_weights_ws(30, 30, 500, 500, 1) == 30 * 30 * 500 * 4 and lib.hk_attn_key_weights_ws(2, 3, 5, 7000, 1) > 2 * 3 * 5 * 4
    assert lib.hk_prefix_attn_ws(2, 2, 1, 8, 4, 64) == lib.hk_decode_attn_weights_ws(2, 2, 128, 5) == L.HK_NO_WS < lib.hk_prefix_attn_ws(2, 2, 1, 1000, 4, 64)
    with pytest.raises(RuntimeError, match="not supported"):
        ops.prefix_attention_ws(2, 2, 1, 8, 0, 64)


def _step(**kw):
    base = dict(q=A, k_cache=2 * A, v_cache=3 * A, key_bias=None, w_in=4 * A, w_out=5 * A, out=6 * A, ws=7 * A, ws_bytes=1 << 20, B=2, H=2, head_dim=64,
                n_keys=9, cache_rows=16, bias_bs=0, bias_hs=0, wi_bs=32, wi_hs=16, wo_bs=32, wo_hs=16)
    base.update(kw)
    return L.load().hk_decode_attn_weights_bf16(C.byref(L.HkStepWeightsDesc(**base)), None)


LONG = dict(cache_rows=1040, wi_bs=2080, wi_hs=1040, wo_bs=2080, wo_hs=1040)      # too long for one launch, which takes no workspace


@pytest.mark.parametrize("kw,text", [
    (dict(w_out=None), "null operand"), (dict(n_keys=17), "bad shape"), (dict(n_keys=0), "bad shape"), (dict(head_dim=32), "bad shape"), (dict(q=A + 2), "aligned"),
    (dict(wo_hs=8), "w_out must not overlap"), (dict(wo_bs=24), "w_out must not overlap"), (dict(wi_bs=-1), "negative"), (dict(w_out=4 * A, wo_bs=64), "one layout"),
    (dict(n_keys=1030, ws_bytes=1 << 10, **LONG), "workspace"), (dict(n_keys=1030, ws=None, **LONG), "workspace"), (dict(w_out=4 * A + 64), "overlaps an input"),
    (dict(out=2 * A), "overlaps an input"), (dict(n_keys=1030, ws=5 * A, **LONG), "overlap")])
def test_decode_attn_weights_refuses(kw, text):
    _refused(_step(**kw), text)


def _weights(**kw):
    base = dict(Q=A, K=2 * A, key_bias=None, w_in=None, w_out=3 * A, ws=4 * A, ws_bytes=1 << 16, B=2, H=2, Nq=4, Nk=9, head_dim=64, causal=1, ldq=128, bsq=512,
                ldk=128, bsk=128 * 9, bias_bs=0, wi_bs=0, wi_hs=0, wo_bs=18, wo_hs=9)
    base.update(kw)
    return L.load().hk_attn_key_weights_bf16(C.byref(L.HkKeyWeightsDesc(**base)), None)


MANY = dict(Nq=500, Nk=500, bsq=64000, bsk=64000, wo_bs=1000, wo_hs=500)      # too many products for one launch, which takes no workspace


@pytest.mark.parametrize("kw,text", [
    (dict(K=None), "null operand"), (dict(Nq=10), "bad shape"), (dict(Nq=0), "bad shape"), (dict(head_dim=256), "bad shape"), (dict(ldq=100), "strides"),
    (dict(Q=A + 4), "aligned"), (dict(wo_hs=8), "w_out must not overlap"), (dict(ws_bytes=63, **MANY), "workspace"), (dict(ws=None, **MANY), "workspace"), (dict(w_in=3 * A, wi_bs=20, wi_hs=10), "one layout"),
    (dict(w_out=A), "overlaps an input"), (dict(ws=3 * A, **MANY), "overlaps the workspace")])
def test_attn_key_weights_refuses(kw, text):
    _refused(_weights(**kw), text)


def _evict(**kw):
    base = dict(K=A, V=2 * A, k_out=3 * A, v_out=4 * A, weight=5 * A, weight_out=6 * A, key_bias=None, key_bias_out=None, kept=7 * A, B=2, H=2, head_dim=64,
                n_keys=9, budget=4, recent=1, ldk=128, bsk=128 * 9, ldv=128, bsv=128 * 9, ldko=128, bsko=512, ldvo=128, bsvo=512, w_bs=18, w_hs=9, wo_bs=8,
                wo_hs=4, b_bs=0, b_hs=0, bo_bs=0, bo_hs=0)
    base.update(kw)
    return L.load().hk_cache_evict_bf16(C.byref(L.HkCacheEvictDesc(**base)), None)


@pytest.mark.parametrize("kw,text", [
    (dict(kept=None), "null operand"), (dict(budget=10), "budget=10"), (dict(budget=0, recent=0), "budget=0"), (dict(recent=5), "recent=5"), (dict(n_keys=0), "n_keys=0"),
    (dict(key_bias=8 * A), "come together"), (dict(ldko=64), "rows must not overlap"), (dict(wo_hs=3), "written must not overlap"), (dict(K=A + 8), "aligned"),
    (dict(k_out=A), "in place together"), (dict(k_out=A, v_out=2 * A, weight_out=5 * A), "one layout"), (dict(v_out=3 * A), "cache each"),
    (dict(k_out=A + 128), "overlaps an input"), (dict(weight_out=5 * A + 4), "overlaps an input"), (dict(kept=3 * A), "two outputs overlap"), (dict(head_dim=100), "bad shape")])
def test_cache_evict_refuses(kw, text):
    _refused(_evict(**kw), text)


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    t = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    w = torch.zeros(1, 2, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.prefix_attention(t, t[0], t[0], t, t)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.attn_key_weights(t, t)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.decode_attn_weights(t.view(1, 128), t.view(1, 1, 128), t.view(1, 1, 128), 1, 2, 64, w)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.cache_evict(t, t, w, 1, 1)
    with pytest.raises(RuntimeError, match="head size"):
        ops.prefix_attention(t[..., :32], t[0], t[0], t, t)
    with pytest.raises(RuntimeError, match="own keys"):
        ops.prefix_attention(t.expand(1, 2, 2, 64), t[0], t[0], t, t)
    with pytest.raises(RuntimeError, match="budget"):
        ops.cache_evict(t, t, w, 1, 2)


# keys too many for one launch, too few for chunks, and so few rows that their sums' bytes are few
@pytest.mark.parametrize("B,H,Nq,Nk", [(1, 4, 1, 400), (2, 2, 1, 400), (1, 1, 4, 385), (1, 4, 1, 448), (1, 1, 1, 385), (1, 5, 1, 400), (4, 1, 1, 430)])
def test_attn_key_weights_of_few_rows_need_their_workspace(B, H, Nq, Nk):
    need = L.load().hk_attn_key_weights_ws(B, H, Nq, Nk, 1)
    assert need != L.HK_NO_WS and need >= 4 * B * H * Nq
    row = H * 64
    kw = dict(B=B, H=H, Nq=Nq, Nk=Nk, ldq=row, bsq=row * Nq, ldk=row, bsk=row * Nk, wo_bs=H * Nk, wo_hs=Nk)
    _refused(_weights(ws=None, **kw), "workspace")
    _refused(_weights(ws_bytes=need - 1, **kw), "workspace")
    _refused(_weights(ws=3 * A, ws_bytes=need, **kw), "overlaps the workspace")


def test_no_real_workspace_has_the_size_that_stands_for_none():
    lib = L.load()
    for B in (1, 2, 3, 8):
        for H in (1, 2, 4, 5):
            for Nq in (1, 2, 4, 33):
                for Nk in (33, 384, 385, 400, 448, 449, 1000, 1500, 5000):
                    row, few = H * 64, lib.hk_attn_key_weights_ws(B, H, Nq, Nk, 1) == L.HK_NO_WS
                    assert few == (Nk <= 384), (B, H, Nq, Nk)
                    if not few:
                        _refused(_weights(ws=None, B=B, H=H, Nq=Nq, Nk=Nk, ldq=row, bsq=row * Nq, ldk=row, bsk=row * Nk, wo_bs=H * Nk, wo_hs=Nk), "workspace")


@pytest.mark.parametrize("call,kw,text", [          # rows of different sequences (or tokens) that share elements, though each stride alone holds a row
    (_prefix, dict(Nq=3, ldo=128, bso=128), "rows must not overlap"), (_prefix, dict(Nq=3, ldo=256, bso=384), "rows must not overlap"),
    (_evict, dict(bsko=128), "rows must not overlap"), (_evict, dict(bsvo=384), "rows must not overlap"), (_evict, dict(B=3, ldko=256, bsko=128), "rows must not overlap"),
    (_evict, dict(k_out=A, v_out=2 * A, weight_out=5 * A, ldko=128, bsk=128 * 4, bsko=128 * 4, bsvo=128 * 9, wo_bs=18, wo_hs=9), "rows must not overlap"),
    (_step, dict(wo_hs=16, wo_bs=16), "w_out must not overlap"), (_weights, dict(wo_hs=9, wo_bs=9), "w_out must not overlap"),
    (_evict, dict(wo_bs=4, wo_hs=4), "written must not overlap"), (_evict, dict(key_bias=8 * A, key_bias_out=9 * A, b_bs=18, b_hs=9, bo_bs=4, bo_hs=4), "written must not overlap")])
def test_outputs_whose_rows_share_elements_are_refused(call, kw, text):
    _refused(call(**kw), text)


KV = dict(K=A, V=A + 256, ldk=256, bsk=256 * 9, ldv=256, bsv=256 * 9)                              # [B, 9, 2, 2, 64]: rows of 256 bytes, side by side
SAME = dict(k_out=A, v_out=A + 256, weight_out=5 * A, ldko=256, bsko=256 * 9, ldvo=256, bsvo=256 * 9, wo_bs=18, wo_hs=9)


@pytest.mark.parametrize("kw,text", [               # interleaved, and a piece into each other; interleaved with another period
    (dict(KV, **dict(SAME, v_out=A + 240, V=A + 240)), "an output overlaps an input"), (dict(KV, **dict(SAME, V=A + 272, v_out=A + 272)), "an output overlaps an input"),
    (dict(KV, **dict(SAME, ldv=264, bsv=264 * 9, ldvo=264, bsvo=264 * 9)), "an output overlaps an input"), (dict(KV, k_out=A + 128, ldko=256, bsko=256 * 9), "an output overlaps an input"),
    (dict(KV, **dict(SAME, bsv=256 * 9 + 128, bsvo=256 * 9 + 128)), "an output overlaps an input"), (dict(k_out=3 * A, v_out=3 * A + 128, ldko=256, ldvo=256, bsko=1024, bsvo=1024), "two outputs overlap"),
    (dict(KV, k_out=A + 512 * 18 - 256, v_out=4 * A, ldko=256, bsko=1024), "an output overlaps an input"),
    (dict(k_out=3 * A, v_out=3 * A + 128 * 2 * 3, bsko=1024, bsvo=1024), "two outputs overlap")])
def test_interleaved_caches_that_meet_are_refused(kw, text):
    _refused(_evict(**kw), text)
