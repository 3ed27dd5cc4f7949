"""8-bit caches and eviction, what needs no GPU: refusals of the C ABI and of the wrappers, workspace sizes, the oracle's own pins."""
import ctypes as C

import pytest
import torch

from oracle import cache8 as ref
from triton_amd import _lib, modules, ops

# (addresses here are made up: with a GPU, a refusal that is missing would launch on them)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="refusals that are made without a GPU")
P = 1 << 20       # an aligned address that no call here gets as far as using


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _cache(**kw):
    c = _lib.Cache8()
    d = dict(k=P, v=P, k_scale=P, v_scale=P, batch=2, n_kv_heads=2, capacity=128, head_dim=64, block=64, k_stride_b=2 * 128 * 64, k_stride_h=128 * 64, k_stride_s=64,
             v_stride_b=2 * 128 * 64, v_stride_h=128 * 64, v_stride_s=64, ks_stride_b=4, ks_stride_h=2, vs_stride_b=4, vs_stride_h=2)
    for n, x in {**d, **kw}.items():
        setattr(c, n, x)
    return c


def _name(lib, st):
    return lib.trn_status_name(st).decode()


def _append(lib, k=P, v=P, tokens=1, strides=(128, 64, 64, 128, 64, 64), **kw):
    return _name(lib, lib.trn_cache8_append_f16(C.byref(_cache(**kw)), k, v, tokens, *strides, None))


def test_append_statuses(lib):
    assert _append(lib, tokens=0) == "TRN_OK" and _append(lib, batch=0) == "TRN_OK" and _append(lib, capacity=0) == "TRN_OK"
    assert _name(lib, lib.trn_cache8_append_f16(None, P, P, 1, *[64] * 6, None)) == "TRN_E_NULL"
    for kw in (dict(k=None), dict(v=None), dict(k_scale=None)):
        assert _append(lib, **kw) == "TRN_E_NULL"
    assert _append(lib, tokens=-1) == "TRN_E_SHAPE" and _append(lib, n_kv_heads=0) == "TRN_E_SHAPE" and _append(lib, batch=-1) == "TRN_E_SHAPE"
    for kw in (dict(head_dim=96), dict(block=48), dict(block=256), dict(capacity=1 << 27), dict(k_stride_s=(1 << 24) + 16)):
        assert _append(lib, **kw) == "TRN_E_UNSUPPORTED"
    assert _append(lib, k_stride_s=48) == "TRN_E_STRIDE" and _append(lib, v_stride_h=0) == "TRN_E_STRIDE" and _append(lib, ks_stride_b=0) == "TRN_E_STRIDE"
    assert _append(lib, k=P + 8) == "TRN_E_ALIGN" and _append(lib, k_stride_h=128 * 64 + 8) == "TRN_E_ALIGN" and _append(lib, strides=(128, 64, 68, 128, 64, 64)) == "TRN_E_ALIGN"
    assert _append(lib, v_scale=P + 2) == "TRN_E_ALIGN"
    assert _append(lib, tokens=1 << 26, capacity=1 << 26, batch=16) == "TRN_E_SHAPE"


def test_append_to_keys_and_values_of_one_place(lib):
    """One tensor for both, or for both their scales, is refused; packed into one tensor, by sequence, head or token, they are a launch (which fails here)."""
    M = 1 << 20
    apart = dict(v=P + M, cache_v=P + 2 * M, k_scale=P + 3 * M, v_scale=P + 4 * M)

    def call(cache_v, v, **kw):
        st = lib.trn_cache8_append_f16(C.byref(_cache(v=cache_v, **kw)), P + 5 * M, v, 1, 128, 64, 64, 128, 64, 64, None)
        return _name(lib, st)
    assert call(**apart) == "TRN_E_LAUNCH"
    for kw in (dict(cache_v=P), dict(cache_v=P + 64 * 127), dict(v_scale=P + 3 * M), dict(v_scale=P + 3 * M + 4)):
        assert call(**{**apart, **kw}) == "TRN_E_UNSUPPORTED", kw
    S, D = 128, 64
    for b, h, s, off in ((4 * S * D, S * D, D, 2 * S * D), (4 * S * D, 2 * S * D, D, S * D), (4 * S * D, D, 4 * D, 2 * D)):
        kw = dict(k_stride_b=b, k_stride_h=h, k_stride_s=s, v_stride_b=b, v_stride_h=h, v_stride_s=s)
        assert call(**{**apart, "cache_v": P + off}, **kw) == "TRN_E_LAUNCH" and call(**{**apart, "cache_v": P + off - 16}, **kw) == "TRN_E_UNSUPPORTED"
    assert call(**{**apart, "v_scale": P + 3 * M + 8}, ks_stride_b=8, ks_stride_h=4, vs_stride_b=8, vs_stride_h=4) == "TRN_E_LAUNCH"


def _attend(lib, q=P, o=P, Hq=4, Sq=1, scale=1.0, w_in=None, w_out=None, ws=None, nbytes=0, qs=(256, 64, 64), os=(256, 64, 64), **kw):
    return _name(lib, lib.trn_cache8_attn_f16(C.byref(_cache(**kw)), q, o, Hq, Sq, *qs, *os, scale, 1, None, w_in, w_out, ws, nbytes, None))


def test_attention_statuses(lib):
    assert _attend(lib, Sq=0) == "TRN_OK" and _attend(lib, batch=0) == "TRN_OK"
    assert _attend(lib, q=None) == "TRN_E_NULL" and _attend(lib, o=None) == "TRN_E_NULL" and _attend(lib, w_in=P) == "TRN_E_NULL"
    assert _attend(lib, Hq=3) == "TRN_E_SHAPE" and _attend(lib, Hq=0) == "TRN_E_SHAPE" and _attend(lib, Sq=-1) == "TRN_E_SHAPE"
    for s in (0.0, -1.0, float("nan")):
        assert _attend(lib, scale=s) == "TRN_E_SHAPE"
    assert _attend(lib, q=P + 8) == "TRN_E_ALIGN" and _attend(lib, o=P + 4) == "TRN_E_ALIGN" and _attend(lib, qs=(256, 60, 64)) == "TRN_E_ALIGN"
    assert _attend(lib, ws=P + 64, nbytes=1 << 30) == "TRN_E_ALIGN"
    assert _attend(lib, os=(256, 0, 64)) == "TRN_E_STRIDE"
    assert _attend(lib, w_out=P) == "TRN_E_SCRATCH" and _attend(lib, w_out=P, ws=P, nbytes=16) == "TRN_E_SCRATCH"
    assert _attend(lib, Sq=1 << 26) == "TRN_E_UNSUPPORTED" and _attend(lib, w_in=P, w_out=P + 64, ws=P, nbytes=1 << 30) == "TRN_E_UNSUPPORTED"


def test_weights_of_no_queries_and_of_no_keys(lib):
    """They are launches like others (which fail here): nothing else would bring the old weights, or zeros, into weights_out.  A cache without keys has no weights
    and needs no workspace for them."""
    W = P + (1 << 20)
    assert _attend(lib, Sq=0, w_out=W) == "TRN_E_LAUNCH" and _attend(lib, Sq=0, w_in=P, w_out=W) == "TRN_E_LAUNCH"
    assert _attend(lib, Sq=0, w_in=W, w_out=W) == "TRN_OK" and _attend(lib, Sq=0, w_out=W, capacity=0) == "TRN_OK"
    assert _attend(lib, Sq=0, w_in=P) == "TRN_E_NULL" and _attend(lib, Sq=0, w_in=P, w_out=P + 64) == "TRN_E_UNSUPPORTED"
    assert _attend(lib, w_out=W, capacity=0) == "TRN_E_LAUNCH"
    assert lib.trn_cache8_attn_workspace_bytes(C.byref(_cache(capacity=0)), 4, 1, 1) == 0


def test_attention_of_more_threads_than_32_bits_number(lib):
    """Refused before the first launch, whichever of the launches it is; one workgroup fewer is a launch (which fails here)."""
    big = dict(ws=P, nbytes=1 << 60)
    assert _attend(lib, batch=1 << 23) == "TRN_E_SHAPE" and _attend(lib, batch=(1 << 23) - 1) == "TRN_E_LAUNCH"                       # the attention's: heads
    assert _attend(lib, batch=1 << 13, Hq=2, Sq=1 << 15) == "TRN_E_LAUNCH" and _attend(lib, batch=1 << 16, Hq=2, Sq=1 << 15) == "TRN_E_SHAPE"      # ... rows
    many = dict(Hq=2, Sq=16, w_out=P + (1 << 20), **big)
    assert _attend(lib, batch=1 << 15, capacity=(1 << 16) + 1, **many) == "TRN_E_SHAPE" and _attend(lib, batch=1 << 15, capacity=1 << 15, **many) == "TRN_E_LAUNCH"      # key weights of many rows
    few = dict(w_out=P + (1 << 20), **big)
    assert _attend(lib, batch=1 << 15, capacity=1 << 18, **few) == "TRN_E_SHAPE" and _attend(lib, batch=1 << 15, capacity=1 << 17, **few) == "TRN_E_LAUNCH"      # ... of few


def test_attention_workspace_is_bounded(lib):
    """By what the shares, the rows' sums and either the scores of few rows or the chunks' sums of many take, whatever the sizes."""
    for B in (1, 3, 32):
        for hkv, g in ((8, 4), (1, 71), (16, 1)):
            for S in (1, 31, 1000, 8192, 131072, 1 << 26):
                for M in (1, 16, 500):
                    for w in (0, 1):
                        c = _cache(batch=B, n_kv_heads=hkv, capacity=S, head_dim=128)
                        n = lib.trn_cache8_attn_workspace_bytes(C.byref(c), hkv * g, M, w)
                        rows = B * hkv * g * M * 4 + 256
                        assert 0 <= n <= 1024 * 32 * 130 * 4 + 1024 + w * (rows + 64 * B * hkv * (S + 32) + (2 << 20)), (B, hkv, g, S, M, w, n)
    assert lib.trn_cache8_attn_workspace_bytes(None, 1, 1, 0) == 0


def _evict(lib, ptrs=None, ws=P, nbytes=1 << 40, **kw):
    e = _lib.CacheEvictDesc()
    d = dict(batch=1, n_kv_heads=2, n_weight_rows=4, keys=64, head_dim=64, code_bytes=2, block=0, keep=16, recent=4, weights_half=0)
    for n, x in {**d, **{k: v for k, v in kw.items() if k in d}}.items():
        setattr(e, n, x)
    for n in ("k_stride", "v_stride"):
        setattr(e, n, (C.c_int64 * 3)(*kw.get(n, (8192, 4096, 64))))
    for n in ("k_out_stride", "v_out_stride"):
        setattr(e, n, (C.c_int64 * 3)(*kw.get(n, (2048, 1024, 64))))
    M = 1 << 20
    p = dict(k=P, v=P + M, k_out=P + 2 * M, v_out=P + 3 * M, ks=None, vs=None, kso=None, vso=None, w=P + 4 * M, wo=None, lengths=None, kept=P + 5 * M, new=None)
    p.update(ptrs or {})
    return _name(lib, lib.trn_cache_evict(C.byref(e), *p.values(), ws, nbytes, None))


def test_evict_statuses(lib):
    assert _evict(lib, batch=0) == "TRN_OK"
    for n in ("k", "v", "k_out", "v_out", "w", "kept"):
        assert _evict(lib, {n: None}) == "TRN_E_NULL"
    assert _evict(lib, ws=None) == "TRN_E_NULL" and _evict(lib, code_bytes=1, block=64) == "TRN_E_NULL"
    for kw in (dict(keep=0), dict(recent=17), dict(recent=-1), dict(n_weight_rows=3), dict(keys=0), dict(n_kv_heads=0)):
        assert _evict(lib, **kw) == "TRN_E_SHAPE"
    for kw in (dict(code_bytes=4), dict(head_dim=80), dict(code_bytes=1, block=48), dict(keys=1 << 27)):
        assert _evict(lib, **kw) == "TRN_E_UNSUPPORTED"
    assert _evict(lib, nbytes=100) == "TRN_E_SCRATCH"
    assert _evict(lib, batch=1 << 22) == "TRN_E_SHAPE" and _evict(lib, batch=1 << 20, n_weight_rows=8) == "TRN_E_SHAPE"      # more threads than 32 bits number
    assert _evict(lib, {"k": P + 8}) == "TRN_E_ALIGN" and _evict(lib, ws=P + 16) == "TRN_E_ALIGN" and _evict(lib, k_stride=(8192, 4096, 68)) == "TRN_E_ALIGN"
    assert _evict(lib, {"k_out": P}) == "TRN_E_STRIDE"                      # the same cache with other strides
    assert _evict(lib, {"k_out": P + 1024}) == "TRN_E_UNSUPPORTED"          # a part of it
    assert _evict(lib, {"v_out": P + 128}) == "TRN_E_UNSUPPORTED" and _evict(lib, {"wo": P + 4 * (1 << 20) + 64}) == "TRN_E_UNSUPPORTED"
    assert _evict(lib, {"v_out": P + 2 * (1 << 20)}) == "TRN_E_UNSUPPORTED"      # both results in one place
    assert _evict(lib, k_stride=(-8192, 4096, 64)) == "TRN_E_STRIDE" and _evict(lib, k_out_stride=(2048, 0, 64)) == "TRN_E_STRIDE"


def test_evict_of_caches_packed_into_one_tensor(lib):
    """Keys and values of one tensor that share no element, in place and into such a tensor: by sequence, by head, and by token, are launches (which fail here); a row
    of one that lies in the other is refused, wherever it is."""
    B, H, S, D = 2, 2, 64, 64
    row = 2 * D      # bytes
    for strides, off in (((2 * H * S * D, S * D, D), H * S * row), ((2 * H * S * D, 2 * S * D, D), S * row), ((2 * H * S * D, D, 2 * H * D), H * row), ((2 * H * S * D, 2 * D, 2 * H * D), row)):
        kw = dict(batch=B, k_stride=strides, v_stride=strides)
        same = dict(k_out_stride=strides, v_out_stride=strides)
        assert _evict(lib, dict(k=P, v=P + off, k_out=P, v_out=P + off), **kw, **same) == "TRN_E_LAUNCH", strides
        Q = P + (1 << 21)
        assert _evict(lib, dict(k=P, v=P + off, k_out=Q, v_out=Q + off), **kw, **same) == "TRN_E_LAUNCH"
        assert _evict(lib, dict(k=P, v=P + off, k_out=Q, v_out=Q), **kw, **same) == "TRN_E_UNSUPPORTED"
        assert _evict(lib, dict(k=P, v=P + off, k_out=P, v_out=P + off - 16), **kw, **same) == "TRN_E_UNSUPPORTED"
        assert _evict(lib, dict(k=P, v=P + off, k_out=P + off, v_out=Q), **kw, **same) == "TRN_E_UNSUPPORTED"          # K's rows to where V's are
        assert _evict(lib, dict(k=P, v=P + off, k_out=P + 32 * strides[2] * 2, v_out=Q), **kw, **same) == "TRN_E_UNSUPPORTED"


def test_evict_of_scales_that_share_memory(lib):
    """Scale outputs of two heads, or of keys and values, in one place are refused; apart, over their inputs and packed into one tensor they are launches (which
    fail here)."""
    M = 1 << 20

    def call(ks=P + 6 * M, vs=P + 7 * M, kso=P + 8 * M, vso=P + 9 * M, k=(4, 2), v=(4, 2), ko=(2, 1), vo=(2, 1)):
        e = _lib.CacheEvictDesc(batch=2, n_kv_heads=2, n_weight_rows=4, keys=64, head_dim=64, code_bytes=1, block=32, keep=16, recent=4)
        e.k_stride = e.v_stride = (8192, 4096, 64)
        e.k_out_stride = e.v_out_stride = (2048, 1024, 64)
        e.k_scale_stride, e.v_scale_stride, e.k_scale_out_stride, e.v_scale_out_stride = k, v, ko, vo
        return _name(lib, lib.trn_cache_evict(C.byref(e), P, P + M, P + 2 * M, P + 3 * M, ks, vs, kso, vso, P + 4 * M, None, None, P + 5 * M, None, P, 1 << 40, None))
    assert call() == "TRN_E_LAUNCH" and call(kso=P + 6 * M, vso=P + 7 * M, ko=(4, 2), vo=(4, 2)) == "TRN_E_LAUNCH"
    for kw in (dict(ko=(0, 1)), dict(ko=(2, 0)), dict(vo=(0, 1)), dict(vo=(2, 0)), dict(k=(-4, 2)), dict(vo=(2, -1))):
        assert call(**kw) == "TRN_E_STRIDE", kw
    for kw in (dict(ks=P + 6 * M + 2), dict(vs=P + 1), dict(kso=P + 8 * M + 2), dict(vso=P + 9 * M + 3)):
        assert call(**kw) == "TRN_E_ALIGN", kw
    for kw in (dict(vso=P + 8 * M), dict(vso=P + 8 * M + 4), dict(vso=P + 8 * M + 4, ko=(4, 1), vo=(4, 1))):
        assert call(**kw) == "TRN_E_UNSUPPORTED", kw
    assert call(vso=P + 8 * M + 8, ko=(4, 1), vo=(4, 1)) == "TRN_E_LAUNCH" and call(vso=P + 8 * M + 4, ko=(4, 2), vo=(4, 2)) == "TRN_E_LAUNCH"      # by sequence, by head


def test_wrappers_refuse_cpu_tensors_and_bad_constants():
    t = torch.zeros(1, 2, 64, 64, dtype=torch.float16)
    c = torch.zeros(1, 2, 64, 64, dtype=torch.uint8)
    s = torch.zeros(1, 2, 1)
    with pytest.raises(ValueError):
        ops.cache8_append(t, t, c, c, s, s)
    with pytest.raises(ValueError):
        ops.cache8_attention(t, c, c, s, s, t)
    with pytest.raises(ValueError):
        ops.cache_evict(t, t, torch.zeros(1, 2, 64), t, t, torch.zeros(1, 2, 8, dtype=torch.int32), 8, 1, c)
    for kw in (dict(keep=0), dict(keep=4, recent=5), dict(keep=4, recent=-1)):
        with pytest.raises(ValueError):
            modules.get("evict", "cache", **kw)
    with pytest.raises(TypeError):
        modules.get("attn8", "cache").forward(c, s)
    with pytest.raises(KeyError):
        modules.get("attn4", "cache")
    with pytest.raises(KeyError):
        modules.get("roco", "cache8", head_dim=64)


def test_oracle_codes_against_the_type():
    x = torch.randn(20000, generator=torch.Generator().manual_seed(1)) * torch.exp(3 * torch.randn(20000, generator=torch.Generator().manual_seed(2)))
    x = x[x.abs() < 464]
    assert torch.equal(ref.encode(x), x.to(torch.float8_e4m3fn).view(torch.uint8))
    middle = (ref.VALUES[:126] + ref.VALUES[1:127]) / 2
    assert torch.equal(ref.encode(middle), middle.float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(torch.nan_to_num(ref.VALUES, nan=1e9), torch.nan_to_num(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double(), nan=1e9))
    assert ref.scale_for(torch.tensor([448.0])) == 1.0 and ref.scale_for(torch.tensor([448.5])) == 2.0 and ref.scale_for(torch.tensor([0.0])) == ref.FLOOR


def test_oracle_attention_against_the_whole_softmax():
    g = torch.Generator().manual_seed(4)
    q = torch.randn(1, 2, 3, 64, generator=g).half()
    k8, v8 = (ref.encode(torch.randn(1, 1, 40, 64, generator=g) * 50) for _ in range(2))
    s = torch.full((1, 1, 2), 0.03125)
    o, lse, w, *_ = ref.attention(q, k8, v8, s, s, 0.125, False, [40], [3], 32)
    k, v = ref.decode(k8) * 0.03125, ref.decode(v8) * 0.03125
    p = torch.softmax(q.double() @ k.transpose(2, 3) * 0.125, -1)
    assert torch.allclose(o, p @ v) and torch.allclose(w, p.sum((1, 2))[:, None]) and torch.allclose(lse.exp(), torch.exp(q.double() @ k.transpose(2, 3) * 0.125).sum(-1))
