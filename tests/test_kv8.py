"""CPU checks of the paged 8-bit cache: refusals of the C entry points before any device work, the workspace query, the checks
of the Python binding, and the arithmetic of the tests' own plain form."""
import ctypes

import numpy as np
import pytest
import torch

import dgx_attn as A
import kv8_ref as R

INVALID, PTR = 1, 1 << 20            # a pointer that no refused call may follow


def cache(**kw):
    d = dict(K=PTR, V=PTR, Ks=PTR, Vs=PTR, pages=10, page=64, NKV=4, HD=256)
    d.update(kw)
    return A._KV8(**d)


def attn(c=None, **kw):
    d = dict(Q=PTR, q=1, table=PTR, stride=20, O=PTR, o=1, lse=None, B=2, T=1, rows=2, NQ=24, ctx=PTR, cu=PTR, anc=None, max_pos=600,
             chunk=0, ws=PTR, ws_bytes=1 << 40, scale=0.0, window=0)
    d.update(kw)
    c = cache() if c is None else c
    return A.lib().dgx_attn_kv8(d["Q"], d["q"], ctypes.addressof(c) if c else None, d["table"], d["stride"], d["O"],
                                d["o"], d["lse"], d["B"], d["T"], d["rows"], d["NQ"], d["ctx"], d["cu"], d["anc"], d["max_pos"],
                                d["chunk"], d["ws"], d["ws_bytes"], None, d["scale"], d["window"])


@pytest.mark.parametrize("kw", [dict(Q=None), dict(O=None), dict(table=None), dict(ctx=None), dict(q=0), dict(q=3), dict(o=3), dict(o=-1),
                                dict(B=-1), dict(T=-1), dict(rows=-1), dict(NQ=0), dict(NQ=23), dict(max_pos=-1), dict(max_pos=1 << 30),
                                dict(chunk=-64), dict(chunk=32), dict(chunk=100), dict(chunk=(1 << 20) + 64), dict(stride=9),
                                dict(Q=PTR + 8), dict(O=PTR + 2), dict(ws=PTR + 4), dict(cu=None, rows=3), dict(anc=PTR, T=33, rows=66),
                                dict(ws=None, chunk=64), dict(ws_bytes=100, chunk=64), dict(B=1, T=1 << 29, rows=1 << 29, NQ=4, max_pos=(1 << 30) - 1, chunk=64, stride=1 << 24), dict(B=1 << 20, T=1 << 20), dict(NQ=4 * 16384)])
def test_attention_refuses(kw):
    assert attn(**kw) == INVALID


@pytest.mark.parametrize("kw", [dict(K=None), dict(V=None), dict(Ks=None), dict(Vs=None), dict(pages=0), dict(page=8), dict(page=48),
                                dict(page=128), dict(NKV=0), dict(HD=64), dict(HD=192), dict(K=PTR + 8), dict(V=PTR + 1), dict(pages=1 << 26)])
def test_a_cache_that_is_none_is_refused(kw):
    c = cache(**kw)
    assert attn(c) == INVALID
    assert A.lib().dgx_kv8_append(PTR, PTR, 2, 1024, 1024, ctypes.addressof(c), PTR, 3, None) == INVALID


def test_null_cache_is_refused():
    assert attn(0) == INVALID
    assert A.lib().dgx_kv8_append(PTR, PTR, 2, 1024, 1024, None, PTR, 3, None) == INVALID


def test_nothing_to_do_is_no_error():
    for kw in (dict(B=0), dict(T=0), dict(rows=0)):
        assert attn(**kw) == 0
    c = cache()
    assert A.lib().dgx_kv8_append(None, None, 2, 1024, 1024, ctypes.addressof(c), None, 0, None) == 0


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(slots=None), dict(dt=3), dict(rows=-1), dict(ks=1016), dict(vs=1000), dict(ks=1025),
                                dict(vs=1028), dict(k=PTR + 8), dict(v=PTR + 2)])
def test_append_refuses(kw):
    d = dict(k=PTR, v=PTR, dt=2, ks=1024, vs=1024, slots=PTR, rows=4)
    d.update(kw)
    c = cache()
    assert A.lib().dgx_kv8_append(d["k"], d["v"], d["dt"], d["ks"], d["vs"], ctypes.addressof(c), d["slots"], d["rows"], None) == INVALID


@pytest.mark.parametrize("kw", [dict(ctx=None), dict(add=None), dict(B=-1), dict(page=24), dict(page=0), dict(page=128), dict(table=None),
                                dict(stride=3), dict(cols=-1), dict(free=None), dict(cap=-1), dict(fin=None), dict(fout=None), dict(cu=None),
                                dict(slots=None), dict(rows=-1), dict(status=None)])
def test_plan_refuses(kw):
    d = dict(ctx=PTR, add=PTR, B=3, page=64, table=PTR, stride=4, cols=4, free=PTR, cap=9, fin=PTR, fout=PTR, cu=PTR, slots=PTR, rows=5, status=PTR)
    d.update(kw)
    assert A.lib().dgx_kv8_plan(d["ctx"], d["add"], d["B"], d["page"], d["table"], d["stride"], d["cols"], d["free"], d["cap"], d["fin"],
                                d["fout"], d["cu"], d["slots"], d["rows"], d["status"], None) == INVALID


def test_workspace_holds_the_partials():
    for B, T, NQ, NKV, HD, mp, chunk in ((16, 1, 24, 4, 256, 8191, 512), (1, 1, 16, 1, 512, 131071, 0), (3, 8, 16, 8, 128, 5000, 64), (2, 300, 16, 8, 256, 4000, 1024)):
        n = A.attn_kv8_workspace(B, T, B * T, NQ, NKV, HD, mp, chunk)
        if chunk:
            assert n >= B * T * NQ * (mp // chunk + 1) * (HD + 2) * 4
    assert A.attn_kv8_workspace(2, 1, 2, 16, 4, 128, 63, 64) == 0
    for bad in (dict(NQ=7), dict(HD=100), dict(max_pos=1 << 30), dict(chunk=65)):
        d = dict(B=1, T=1, rows=1, NQ=8, NKV=4, HD=128, max_pos=100, chunk=0)
        d.update(bad)
        with pytest.raises(ValueError):
            A.attn_kv8_workspace(**d)


def test_a_workspace_without_a_tree_holds_one_too():
    """Runs of up to 32 tokens take a tree or not from step to step: the default size fits both."""
    more = 0
    for NQ, NKV, HD in ((24, 4, 256), (16, 1, 512), (16, 4, 128)):
        for B in (1, 5, 16):
            for T in (2, 11, 16, 32):
                for max_pos in (300, 1200, 5000, 12000):
                    both, tree = (A.attn_kv8_workspace(B, T, B * T, NQ, NKV, HD, max_pos, tree=t) for t in (False, True))
                    assert both >= tree
                    more += tree > 0
    assert more


def test_the_binding_refuses_wrong_tensors():
    f8 = torch.float8_e4m3fn
    K, V, S = torch.zeros(3, 2, 16, 128).to(f8), torch.zeros(3, 2, 128, 16).to(f8), torch.ones(3, 2)
    c = A.KV8Cache(K, V, S, S.clone())
    for bad in ((K, K, S, S), (K, V, S[:2], S), (K.float(), V, S, S), (K, V, S.double(), S), (K.transpose(2, 3), V.transpose(2, 3), S, S),
                (torch.zeros(3, 2, 24, 128).to(f8), torch.zeros(3, 2, 128, 24).to(f8), S, S)):
        with pytest.raises(ValueError):
            A.KV8Cache(*bad)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):                        # host tensors
        A.kv8_append(torch.zeros(2, 2, 128), torch.zeros(2, 2, 128), c, i)
    with pytest.raises(ValueError):
        A.attn_kv8(torch.zeros(2, 4, 128).half(), c, torch.zeros(2, 3, dtype=torch.int32), i, torch.zeros(2, 4, 128).half(), 1, 20)
    with pytest.raises(ValueError):
        A.kv8_plan(i, i, 16, torch.zeros(2, 3, dtype=torch.int32), i, i[:1], i[:1], torch.zeros(3, dtype=torch.int32), i, i[:1])


CALLER = r"""
#include "dgx_attn.hpp"
#include <cstdio>
int main(int argc, char **) {
    dgx_kv8 c{(void *)16, (void *)16, (float *)16, (float *)16, 8, 64, 4, 256};
    launch_attn_kv8<__half, float>(nullptr, c, nullptr, 0, nullptr, 0, 1, 0, 24, nullptr, nullptr, 100, nullptr, 0);
    launch_attn_kv8<__hip_bfloat16, __hip_bfloat16>(nullptr, c, nullptr, 0, nullptr, 2, 1, 0, 24, nullptr, nullptr, 100, nullptr, 0);
    kv8_append<float>(nullptr, nullptr, 1024, 1024, c, nullptr, 0);
    printf("%d %d\n", attn_kv8_workspace(1, 1, 1, 24, 4, 256, 63) == 0, attn_kv8_workspace(16, 1, 16, 24, 4, 256, 8191) > 0);
    fflush(stdout);
    if (argc > 1) kv8_plan(nullptr, nullptr, 1, 48, nullptr, 0, 0, nullptr, 0, nullptr, nullptr, nullptr, nullptr, 0, nullptr);
    return 0;
}
"""


def test_cxx_callers(tmp_path):
    """The C++ names compile, link and run; a refused call ends the process with its name, as the other launchers do."""
    import os
    import signal
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "dgx-serving_amd")
    (tmp_path / "caller.cpp").write_text(CALLER)
    exe = str(tmp_path / "caller")
    cmd = ["/opt/rocm/bin/amdclang++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(root, "include"), "-I", "/opt/rocm/include",
           str(tmp_path / "caller.cpp"), "-o", exe, "-L", lib, "-ldgx_attn", "-L", "/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{lib}:/opt/rocm/lib"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    env = {k: v for k, v in os.environ.items() if not k.startswith("G4_")}
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60, env=env)
    assert out.returncode == 0 and out.stdout.split() == ["1", "1"], out.stderr
    bad = subprocess.run([exe, "x"], capture_output=True, text=True, timeout=60, env=env)
    assert bad.returncode == -signal.SIGABRT and "[kv8_plan] failed" in bad.stderr, (bad.returncode, bad.stderr)


def test_reference_codes_are_torchs():
    """The tests' encoder against torch's cast, and its decoder against torch's values."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(4000) * 100, (R.POSITIVE[:-1] + R.POSITIVE[1:]) / 2, rng.standard_normal(2000) * 0.01]).astype(np.float32)
    x = np.clip(x, -448, 448)
    assert np.array_equal(R.encode(x.astype(np.float64)), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(R.TABLE)) and np.array_equal(t[~np.isnan(t)], R.TABLE[~np.isnan(R.TABLE)])
    for a, e in ((448.0, 0), (448.1, 1), (224.0, -1), (0.0, -40), (1e30, 40)):
        assert R.exponent(a) == e
