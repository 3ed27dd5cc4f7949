"""Operators of the fp16 cache, what needs no GPU: refusals of the C ABI and of the wrappers, structures, workspace sizes, how work is shared out, the oracle's own pins."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from oracle import cache16 as ref
from triton_amd import _lib, modules, ops

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")
# (addresses here are made up: with a GPU, a refusal that is missing would launch on them)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="refusals that are made without a GPU")
P, M = 1 << 24, 1 << 20       # aligned addresses that no call here gets as far as using


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _st(*x):
    return (C.c_int64 * len(x))(*x)


def _cache(**kw):
    c = _lib.Cache16()
    d = dict(k=P, v=P + M, batch=2, n_kv_heads=2, capacity=128, head_dim=64, k_stride=(2 * 128 * 64, 128 * 64, 64), v_stride=(2 * 128 * 64, 128 * 64, 64))
    for n, x in {**d, **kw}.items():
        setattr(c, n, x)
    return c


def _name(lib, st):
    return lib.trn_status_name(st).decode()


ROWS = (4 * 64 * 3, 64, 4 * 64)       # [2, 4, 3, 64] token by token


def _rope(lib, cache=None, q=P + 2 * M, qo=P + 3 * M, k=P + 4 * M, v=P + 5 * M, heads=4, tokens=3, st=(ROWS,) * 4, **kw):
    r = _lib.Rope()
    for n, x in {**dict(inv_freq=P + 6 * M, pairs=32, axes=1, sections=(32, 0, 0, 0), eps=1e-6), **kw}.items():
        setattr(r, n, x)
    return _name(lib, lib.trn_cache_rope_append_f16(C.byref(cache or _cache()), C.byref(r), q, qo, k, v, heads, tokens, *(_st(*s) for s in st), None))


@no_gpu
def test_rope_statuses(lib):
    assert _rope(lib) == "TRN_E_LAUNCH"                                        # all is well, but for the GPU
    assert _rope(lib, tokens=0) == "TRN_OK" and _rope(lib, _cache(batch=0)) == "TRN_OK"
    assert _rope(lib, _cache(capacity=0, k=None, v=None)) == "TRN_E_LAUNCH"    # (queries are turned all the same)
    for kw in (dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(inv_freq=None), dict(axes=2, sections=(16, 16, 0, 0))):
        assert _rope(lib, **kw) == "TRN_E_NULL", kw
    for kw in (dict(tokens=-1), dict(heads=0), dict(sections=(31, 0, 0, 0)), dict(sections=(33, 0, 0, 0)), dict(norm=1, eps=-1.0), dict(norm=1, eps=float("nan"))):
        assert _rope(lib, **kw) == "TRN_E_SHAPE", kw
    for kw in (dict(pairs=30, sections=(30, 0, 0, 0)), dict(pairs=36, sections=(36, 0, 0, 0)), dict(axes=0), dict(axes=5), dict(gamma_q=P + 7 * M)):
        assert _rope(lib, **kw) == "TRN_E_UNSUPPORTED", kw
    for kw in (dict(q=P + 2 * M + 8), dict(inv_freq=P + 4), dict(norm=1, gamma_k=P + 2), dict(st=((4 * 64 * 3, 64, 4 * 64 + 4),) + (ROWS,) * 3)):
        assert _rope(lib, **kw) == "TRN_E_ALIGN", kw
    for kw in (dict(st=((-768, 64, 256),) + (ROWS,) * 3), dict(st=(ROWS, (768, 0, 256), ROWS, ROWS))):
        assert _rope(lib, **kw) == "TRN_E_STRIDE", kw
    for c in (_cache(head_dim=96), _cache(capacity=(1 << 26) + 1), _cache(k_stride=(1 << 30, 128 * 64, (1 << 23) + 8))):
        assert _rope(lib, c) == "TRN_E_UNSUPPORTED"
    assert _rope(lib, _cache(k_stride=(2 * 128 * 64, 128 * 64, 56))) == "TRN_E_STRIDE" and _rope(lib, _cache(v_stride=(2 * 128 * 64, 0, 64))) == "TRN_E_STRIDE"
    assert _rope(lib, _cache(k=P + 8)) == "TRN_E_ALIGN" and _rope(lib, _cache(n_kv_heads=0)) == "TRN_E_SHAPE"


@no_gpu
def test_rope_of_what_shares_memory(lib):
    """q_out may be q; q, k and v may be packed into one tensor, and the caches into another; anything else that shares memory with what is written is refused."""
    packed = (8 * 64 * 3, 64, 8 * 64)                                          # [2, 4 + 2 + 2, 3, 64] token by token
    Q = P + 2 * M
    one = dict(q=Q, k=Q + 4 * 64 * 2, v=Q + 6 * 64 * 2)
    assert _rope(lib, qo=Q, st=(packed,) * 4, **one) == "TRN_E_LAUNCH"
    assert _rope(lib, st=(packed, ROWS, packed, packed), **one) == "TRN_E_LAUNCH"
    assert _rope(lib, qo=Q + 128, st=(packed,) * 4, **one) == "TRN_E_UNSUPPORTED"
    assert _rope(lib, qo=P + 4 * M) == "TRN_E_UNSUPPORTED" and _rope(lib, qo=P + 5 * M) == "TRN_E_UNSUPPORTED"
    assert _rope(lib, k=P) == "TRN_E_UNSUPPORTED" and _rope(lib, v=P + M + 4096) == "TRN_E_UNSUPPORTED" and _rope(lib, qo=P) == "TRN_E_UNSUPPORTED"
    assert _rope(lib, _cache(v=P)) == "TRN_E_UNSUPPORTED"
    both = (4 * 128 * 64, 128 * 64, 64)
    assert _rope(lib, _cache(v=P + 2 * 128 * 64 * 2, k_stride=both, v_stride=both)) == "TRN_E_LAUNCH"


def _prefix(lib, cache=None, q=P + 2 * M, o=P + 3 * M, heads=4, seq=3, st=(ROWS, ROWS), scale=0.125, ws=P + 8 * M, n=1 << 40, **kw):
    p = _lib.Prefix()
    for x, y in {**dict(k=P + 6 * M, v=P + 7 * M, keys=100, k_stride=(100 * 64, 64), v_stride=(100 * 64, 64)), **kw}.items():
        setattr(p, x, y)
    return _name(lib, lib.trn_cache_prefix_attn_f16(C.byref(cache or _cache()), C.byref(p), q, o, heads, seq, _st(*st[0]), _st(*st[1]), scale, 1, ws, n, None))


@no_gpu
def test_prefix_statuses(lib):
    assert _prefix(lib) == "TRN_E_LAUNCH" and _prefix(lib, keys=0, k=None, v=None) == "TRN_E_LAUNCH" and _prefix(lib, _cache(capacity=0, k=None, v=None)) == "TRN_E_LAUNCH"
    assert _prefix(lib, seq=0) == "TRN_OK" and _prefix(lib, _cache(batch=0)) == "TRN_OK"
    for kw in (dict(q=None), dict(o=None), dict(k=None), dict(v=None)):
        assert _prefix(lib, **kw) == "TRN_E_NULL", kw
    for kw in (dict(heads=3), dict(heads=0), dict(seq=-1), dict(keys=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert _prefix(lib, **kw) == "TRN_E_SHAPE", kw
    for kw in (dict(seq=1 << 25), dict(keys=(1 << 26) + 1), dict(k_stride=(1 << 40, (1 << 23) + 8)), dict(o=P + 2 * M), dict(o=P + 128), dict(o=P + M), dict(o=P + 6 * M), dict(o=P + 7 * M + 640)):
        assert _prefix(lib, **kw) == "TRN_E_UNSUPPORTED", kw
    for kw in (dict(q=P + 2 * M + 8), dict(o=P + 3 * M + 4), dict(k=P + 6 * M + 2), dict(ws=P + 128)):
        assert _prefix(lib, **kw) == "TRN_E_ALIGN", kw
    assert _prefix(lib, st=(ROWS, (768, 64, 0))) == "TRN_E_STRIDE" and _prefix(lib, v_stride=(100 * 64, 56)) == "TRN_E_STRIDE"
    # (many keys: shares, and a workspace for them)
    big = _cache(capacity=1 << 16, k_stride=(1 << 23, 1 << 22, 64), v_stride=(1 << 23, 1 << 22, 64), v=P + (1 << 30))
    far = dict(q=P + (1 << 32), o=P + (1 << 33), k=P + (1 << 34), v=P + (1 << 35), seq=1)
    need = lib.trn_cache_prefix_attn_workspace_bytes(C.byref(big), 100, 4, 1)
    assert need > 0 and _prefix(lib, big, n=need, **far) == "TRN_E_LAUNCH"
    assert _prefix(lib, big, n=need - 1, **far) == "TRN_E_SCRATCH" and _prefix(lib, big, ws=None, **far) == "TRN_E_SCRATCH"
    assert lib.trn_cache_prefix_attn_workspace_bytes(None, 1, 1, 1) == 0 and lib.trn_cache_prefix_attn_workspace_bytes(C.byref(big), 100, 3, 1) == 0


def _sparse(lib, cache=None, bounds=P + 6 * M, block=32, top=4, sink=1, recent=1, q=P + 2 * M, o=P + 3 * M, sel=P + 7 * M, heads=4, seq=3, scale=0.125, ws=P + 8 * M, n=1 << 40):
    return _name(lib, lib.trn_cache_sparse_attn_f16(C.byref(cache or _cache()), bounds, block, top, sink, recent, q, o, sel, heads, seq, _st(*ROWS), _st(*ROWS), scale, ws, n, None))


@no_gpu
def test_sparse_and_bounds_statuses(lib):
    assert _sparse(lib) == "TRN_E_LAUNCH" and _sparse(lib, seq=0) == "TRN_OK" and _sparse(lib, _cache(batch=0)) == "TRN_OK"
    assert _sparse(lib, _cache(capacity=0, k=None, v=None), bounds=None) == "TRN_E_LAUNCH"
    for kw in (dict(bounds=None), dict(q=None), dict(o=None), dict(sel=None)):
        assert _sparse(lib, **kw) == "TRN_E_NULL", kw
    for kw in (dict(top=0), dict(sink=-1), dict(recent=0), dict(top=2, sink=1, recent=2), dict(heads=6 + 1), dict(scale=-1.0)):
        assert _sparse(lib, **kw) == "TRN_E_SHAPE", kw
    for kw in (dict(block=48), dict(block=256), dict(top=(1 << 16) + 1), dict(o=P + 64), dict(o=P + 2 * M + 128), dict(sel=P + 3 * M), dict(sel=P + 2 * M + 64), dict(sel=P + 6 * M), dict(o=P + 6 * M), dict(sel=P + 64), dict(sel=P + M)):
        assert _sparse(lib, **kw) == "TRN_E_UNSUPPORTED", kw
    assert _sparse(lib, bounds=P + 6 * M + 8) == "TRN_E_ALIGN" and _sparse(lib, sel=P + 2) == "TRN_E_ALIGN"
    assert lib.trn_cache_sparse_attn_workspace_bytes(C.byref(_cache()), 32, 4, 4, 3) == 0 and _sparse(lib, ws=None) == "TRN_E_LAUNCH"      # four blocks, all selected
    need = lib.trn_cache_sparse_attn_workspace_bytes(C.byref(_cache()), 32, 3, 4, 3)
    assert need > 0 and _sparse(lib, top=3, n=need) == "TRN_E_LAUNCH" and _sparse(lib, top=3, n=need - 1) == "TRN_E_SCRATCH" and _sparse(lib, top=3, ws=None) == "TRN_E_SCRATCH"
    assert lib.trn_cache_sparse_attn_workspace_bytes(C.byref(_cache()), 48, 4, 4, 3) == 0
    bounds = lambda block=32, tokens=1, to=P + 6 * M, **kw: _name(lib, lib.trn_cache_bounds_f16(C.byref(_cache(v=None, **kw)), block, tokens, to, None))
    assert bounds() == "TRN_E_LAUNCH" and bounds(tokens=0) == "TRN_OK" and bounds(capacity=0) == "TRN_OK" and bounds(block=16) == "TRN_E_UNSUPPORTED"
    assert bounds(tokens=-1) == "TRN_E_SHAPE" and bounds(to=None) == "TRN_E_NULL" and bounds(to=P + 6 * M + 4) == "TRN_E_ALIGN" and bounds(to=P) == "TRN_E_UNSUPPORTED"


def test_wrappers_refuse_cpu_tensors_and_bad_constants():
    t, n = torch.zeros(1, 2, 64, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.float64)
    calls = [lambda: ops.cache_rope_append(t, t, t, t, t, t, n), lambda: ops.cache_prefix_attention(t, t, t, t[0], t[0], t),
             lambda: ops.cache_bounds(t, torch.zeros(1, 2, 1, 2, 64, dtype=torch.float16)),
             lambda: ops.cache_sparse_attention(t, t, t, torch.zeros(1, 2, 1, 2, 64, dtype=torch.float16), t, torch.zeros(1, 2, 64, 2, dtype=torch.int32), 2)]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    for form, kw in (("cache", {}), ("cache16", dict(head_dim=64))):
        for bad in (dict(top=0), dict(top=4, sink=4), dict(top=4, sink=-1), dict(top=4, recent=0)):
            with pytest.raises(ValueError):
                modules.get("sparse", form, **{**kw, **bad})
    with pytest.raises(KeyError):
        modules.get("rope", "cache16", head_dim=64)
    with pytest.raises(TypeError):
        modules.get("prefix", "cache").forward(t, t)
    for variant, form in (("rope", "cache"), ("prefix", "cache"), ("bounds", "cache")):
        assert modules.get(variant, form).TENSOR_PARAMS == sorted(modules.get(variant, form).TENSOR_PARAMS)


@pytest.mark.parametrize("name, cls", [("trn_cache16", _lib.Cache16), ("trn_rope", _lib.Rope), ("trn_prefix", _lib.Prefix)])
def test_structures_match_c(tmp_path, name, cls):
    header = os.path.join(os.path.dirname(os.path.dirname(CSRC)), "include", "trinity_hip.h")
    fields = [f[0] for f in cls._fields_]
    (tmp_path / "l.c").write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void){{printf("%zu\\n", sizeof({name}));' +
                                  "".join(f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields) + "return 0;}\n")
    subprocess.run(["gcc", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = [int(x) for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


WALK = r"""
#include <cstdio>
#include <initializer_list>
#include "cache16_rules.h"
using namespace trn;
int main() {
    long bad = 0, plans = 0;
    for (int batch : {1, 2, 5, 16, 64, 300}) for (int kv : {1, 2, 8, 16}) for (int g : {1, 4, 8, 71}) for (int sq : {1, 2, 7, 33, 500, 4000}) for (int d : {64, 128})
    for (int cap : {0, 1, 33, 700, 8192, 140000, 1 << 26}) for (int pre : {0, 1, 64, 1000, 16001, 1 << 26}) {
        if ((long)batch * kv * g * sq > (1 << 26)) continue;
        const PlanPrefix p = plan_prefix(batch, kv, cap, d, pre, kv * g, sq);
        ++plans;
        const int64_t heads = (int64_t)batch * kv;
        bool ok = p.R == g * sq && p.slots >= 1 && (p.slots == 1) == (p.bytes == 0) && (p.nq == 1 || p.nq == 2);
        if (p.one) ok = ok && p.slots == p.ns_p && (int64_t)p.n_rt_p * 128 >= p.R && p.first == heads * p.n_rt_p * p.ns_p && p.second == 0;
        else {
            const int64_t rows_p = (int64_t)batch * p.R;
            ok = ok && p.slots == p.ns_p + p.ns_o && (p.ns_p > 0) == (pre > 0) && (p.ns_o > 0 || cap == 0) && (p.ns_o > 0 || pre > 0) && p.ns_p <= 64 && p.ns_o <= 64;
            ok = ok && (int64_t)p.n_rt_p * (p.wide ? 128 : 16 * p.nq) >= rows_p && (int64_t)p.n_rt_o * 16 * p.nq >= p.R && p.first == (int64_t)kv * p.n_rt_p * p.ns_p && p.second == heads * p.n_rt_o * p.ns_o;
        }
        if (p.short_rt) ok = ok && p.short_rt * 16 >= p.R;
        if (p.slots > 1) ok = ok && p.ml >= heads * p.R * p.slots * d * 4 && p.bytes >= p.ml + heads * p.R * p.slots * 8;
        if (!ok) { if (bad < 5) printf("prefix %d %d %d %d %d %d %d\n", batch, kv, g, sq, d, cap, pre); ++bad; }
    }
    for (int batch : {1, 5, 64}) for (int kv : {1, 8}) for (int g : {1, 4, 71}) for (int sq : {1, 7, 500, 4000}) for (int d : {64, 128}) for (int block : {32, 64, 128})
    for (int cap : {0, 1, 8192, 140000, 1 << 26}) for (int top : {1, 40, 1024, 65536}) {
        if ((long)batch * kv * g * sq > (1 << 26)) continue;
        const PlanSparse p = plan_sparse(batch, kv, cap, d, block, top, kv * g, sq);
        ++plans;
        const int64_t heads = (int64_t)batch * kv;
        if (p.dense) {
            const bool good = p.nb <= top && p.step >= 1 && p.step <= sq && heads * p.step <= 0xffffff && p.bytes == plan_prefix(batch, kv, cap, d, 0, kv * g, sq).bytes;
            if (!good) { if (bad < 5) printf("dense %d %d %d %d %d %d %d %d\n", batch, kv, g, sq, d, block, cap, top); ++bad; }
            continue;
        }
        bool ok = p.nbp >= p.nb && p.nbp % 64 == 0 && p.step >= 1 && p.step <= sq && p.norms >= heads * p.nbp * 4 * p.step && p.o >= p.norms + heads * p.nbp / 16 * 4 && p.n_rt * 16 * p.nq >= g;
        ok = ok && p.ns >= 1 && (!p.rows || p.ns == 1) && (p.ns == 1 ? p.bytes == p.o : p.ml >= p.o + heads * sq * g * p.ns * d * 4 && p.bytes >= p.ml + heads * sq * g * p.ns * 8);
        if (!ok) { if (bad < 5) printf("sparse %d %d %d %d %d %d %d %d\n", batch, kv, g, sq, d, block, cap, top); ++bad; }
    }
    printf("%ld plans, %ld bad\n", plans, bad);
    return bad != 0;
}
"""


def test_plans(tmp_path):
    """Every row has a tile and every slot a share; what is kept per slot fits the workspace; over sizes from nothing to the largest."""
    (tmp_path / "walk.cpp").write_text(WALK)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{CSRC}", str(tmp_path / "walk.cpp"), "-o", str(tmp_path / "walk")], check=True)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_oracle_against_whole_tensors():
    """The oracle's loops against the same written at once, for sequences that all are as long."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, s, 64, generator=g).half() for h, s in ((4, 3), (2, 9), (2, 9)))
    kp, vp = (torch.randn(2, 5, 64, generator=g).half() for _ in range(2))
    o, _ = ref.prefix_attention(q, k, v, kp, vp, torch.zeros_like(q), 0.125, True, [9, 9], [3, 3])
    kk, vv = (torch.cat([p.expand(2, 2, 5, 64), x], 2).double().repeat_interleave(2, 1) for p, x in ((kp, k), (vp, v)))
    t = (q.double() @ kk.transpose(2, 3) * 0.125).masked_fill(torch.arange(14) > torch.arange(11, 14)[:, None], -torch.inf)
    assert torch.allclose(o, torch.softmax(t, -1) @ vv)
    inv = 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    outs, _ = ref.rope(q, k[:, :, :3], v[:, :, :3], q, k, v, inv, [9, 9], [3, 3])
    turn = torch.polar(torch.ones(3, 32, dtype=torch.float64), torch.arange(6, 9)[:, None] * inv)
    z = torch.complex(q.double()[..., :32], q.double()[..., 32:]) * turn
    assert torch.allclose(outs[0], torch.cat([z.real, z.imag], -1)) and torch.equal(outs[2][:, :, 6:], v[:, :, :3].double()) and torch.equal(outs[1][:, :, :6], k[:, :, :6].double())
    # blocks that are all selected: the whole attention
    bnd = ref.bounds(k, torch.zeros(2, 2, 1, 2, 64).half(), 32, [9, 9], [9, 9])
    assert torch.equal(bnd[:, :, 0, 0], k.amin(2)) and torch.equal(bnd[:, :, 0, 1], k.amax(2))
    sel = ref.select(q, bnd, torch.zeros(2, 2, 3, 2, dtype=torch.int32), 32, 2, 0, 1, 2, [9, 9], [3, 3], 9)
    assert torch.equal(sel, torch.tensor([0, -1], dtype=torch.int32).expand(2, 2, 3, 2))
    a, _ = ref.sparse_attention(q, k, v, torch.zeros_like(q), sel, 32, 0.125, [9, 9], [3, 3])
    b, _ = ref.prefix_attention(q, k, v, kp[:, :0], vp[:, :0], torch.zeros_like(q), 0.125, True, [9, 9], [3, 3])
    assert torch.allclose(a, b)
