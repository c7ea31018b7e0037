"""What the policy operators refuse, checked without a GPU: the Python side's errors and the C entries' return
codes (arguments are checked before anything is enqueued), and that header, binding and library agree."""
import ctypes
import os
import re

import pytest

from conftest import ROOT

if not os.path.exists(os.path.join(ROOT, "g1.cu_amd", "build", "libg1env.so")):
    pytest.skip("libg1env.so not built (run __graft_entry__.build())", allow_module_level=True)

import torch  # noqa: E402

import g1nn  # noqa: E402

lib = g1nn.lib


def test_binding_matches_header():
    text = open(os.path.join(ROOT, "include", "g1nn.h")).read()
    names = re.findall(r"^(?:int|long)\s+(g1_nn_\w+)\s*\(", text, re.M)
    assert sorted(names) == sorted(g1nn.SIGNATURES)
    for name in names:
        decl = re.search(r"\b" + name + r"\s*\(([^)]*)\)", text).group(1)
        assert len(g1nn.SIGNATURES[name][1]) == decl.count(",") + 1, name
        assert hasattr(lib, name)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    for call in (lambda: g1nn.rms_norm(x, w), lambda: g1nn.rms_norm_q8(x, w),
                 lambda: g1nn.gated_linear(x, torch.zeros(4, 8), torch.zeros(4, 8)),
                 lambda: g1nn.gated_linear_q8(x.to(torch.int8), w, x, w, x, w),
                 lambda: g1nn.clip_grad_norm([x], 1.0), lambda: g1nn.clip_grad_norm([], 1.0)):
        with pytest.raises(ValueError):
            call()


P = 4096   # an aligned address that nothing reads: every call below is refused first


def _norm(type=0, M=2, K=8, x=P, r=None, w=P, y=P, h=None):
    return lib.g1_nn_rms_norm(type, M, K, x, K, r, K, w, 1e-6, y, h, None, None)


def _gated(type=0, M=2, K=8, F=4, x=P, wg=P, wu=P, act=0, y=P):
    return lib.g1_nn_gated(type, M, K, F, x, K, wg, K, wu, K, None, None, act, y, None)


def test_c_entries_refuse():
    for kw in (dict(type=2), dict(type=-1), dict(M=-1), dict(K=0), dict(K=32769), dict(x=None), dict(w=None),
               dict(y=None), dict(r=P), dict(h=P), dict(x=P + 2), dict(y=P + 1), dict(type=1, x=P + 1)):
        assert _norm(**kw) == -1, kw
    for kw in (dict(type=2), dict(M=-1), dict(M=2 ** 30 + 1), dict(K=0), dict(F=0), dict(K=2 ** 17 + 1), dict(F=2 ** 17 + 1),
               dict(act=4), dict(act=-1), dict(x=None), dict(wg=None), dict(wu=None), dict(y=None), dict(x=P + 2)):
        assert _gated(**kw) == -1, kw
    # no rows: nothing to do, nothing read
    assert _norm(M=0, x=None, y=None) == 0 and _gated(M=0, x=None, y=None) == 0
    q8 = lambda **kw: lib.g1_nn_rms_norm_q8(0, kw.get("M", 2), 8, P, 8, None, 0, P, 1e-6, kw.get("q", P),  # noqa: E731
                                            kw.get("s", P), None, None)
    assert q8(q=None) == -1 and q8(s=None) == -1 and q8(M=0) == 0
    gq8 = lambda **kw: lib.g1_nn_gated_q8(kw.get("type", 0), 2, kw.get("K", 8), 4, P, 8, kw.get("s", P), P, P,  # noqa: E731
                                          P, kw.get("su", P), None, None, kw.get("act", 0), kw.get("y", P), None)
    for kw in (dict(type=3), dict(K=2 ** 17 + 1), dict(s=None), dict(su=None), dict(act=9), dict(y=None), dict(y=P + 2)):
        assert gq8(**kw) == -1, kw
    back = lambda **kw: lib.g1_nn_rms_norm_backward(0, 2, 8, kw.get("dy", P), 8, None, 0, P, 8, kw.get("rstd", P),  # noqa: E731
                                                    P, kw.get("dx", P), P, kw.get("ws", P), None)
    for kw in (dict(dy=None), dict(rstd=None), dict(dx=None), dict(ws=None), dict(dx=P + 2)):
        assert back(**kw) == -1, kw
    gback = lambda **kw: lib.g1_nn_gated_backward(0, 2, 8, 4, P, 8, P, 8, P, 8, None, None, kw.get("act", 0),  # noqa: E731
                                                  kw.get("dy", P), 4, P, P, P, P, P, kw.get("ws", P), None)
    for kw in (dict(dy=None), dict(ws=None), dict(act=7), dict(ws=P + 4), dict(dy=P + 1)):
        assert gback(**kw) == -1, kw


def test_clip_refuses():
    def call(n=1, x=P, xt=0, o=P, ot=0, size=4, norm=P, ws=P, most=1.0, table=True):
        a = lambda t, v: (t * max(n, 1))(*[v] * max(n, 1)) if table else None  # noqa: E731
        return lib.g1_nn_clip(n, a(ctypes.c_void_p, x), a(ctypes.c_int, xt), a(ctypes.c_void_p, o), a(ctypes.c_int, ot),
                              a(ctypes.c_long, size), most, norm, ws, None)
    for kw in (dict(n=-1), dict(table=False), dict(x=None), dict(o=None), dict(xt=2), dict(ot=-1), dict(size=-1),
               dict(size=2 ** 62), dict(norm=None), dict(ws=None), dict(ws=P + 8), dict(most=float("nan")), dict(most=-1.0),
               dict(x=P + 2), dict(o=P + 1, ot=1), dict(ot=1)):
        assert call(**kw) == -1, kw


def test_workspace_sizes():
    assert lib.g1_nn_clip_workspace(0) > 0 and lib.g1_nn_clip_workspace(1000) > lib.g1_nn_clip_workspace(10)
    assert lib.g1_nn_rms_norm_backward_workspace(0, 0, 8) >= 0
    assert lib.g1_nn_gated_backward_workspace(0, 0, 8, 8) >= 0
    # sizes in 64 bits
    assert lib.g1_nn_gated_backward_workspace(0, 2 ** 22, 512, 4096) > 2 ** 32


def test_kernels_hold_their_values_in_registers():
    """From the compiler's report that build() records beside the library: no kernel of the operators has scratch, but
    the norm's gradients of rows longer than 8192 fp32 or 16384 bf16 values, whose registers do not hold a row three
    times; and the gated block's large tiles leave room for two blocks on a CU."""
    import json
    res = {f: r for f, r in json.load(open(os.path.join(ROOT, "g1.cu_amd", "build", "resource_usage.json"))).items()
           if "4g1nn" in f}
    assert len(res) > 40
    for f, r in res.items():
        if "k_rms_norm_grad" in f and "Li1024E" in f:
            continue
        assert r["ScratchSize"] == 0 and r["VGPRs Spill"] == 0, (f, r)
        if "k_gated" in f:
            assert r["Occupancy"] >= 2, (f, r)
