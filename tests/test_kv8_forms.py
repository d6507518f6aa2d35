"""CPU checks of the query for the form that a call over the paged 8-bit cache takes."""
import ctypes

import numpy as np
import pytest

import dgx_attn as A
import test_kv8_forms_gpu as G


@pytest.mark.parametrize("kw", [dict(B=-1), dict(T=-1), dict(rows=-1), dict(NQ=7), dict(NKV=0), dict(HD=64), dict(max_pos=-1), dict(max_pos=1 << 30),
                                dict(chunk=65), dict(chunk=-64)])
def test_the_form_of_refused_sizes_is_refused(kw):
    d = dict(B=2, T=3, rows=6, NQ=8, NKV=4, HD=128, max_pos=100, chunk=0)
    assert A.attn_kv8_form(**d)[0] == 0
    with pytest.raises(ValueError):
        A.attn_kv8_form(**dict(d, **kw))
    assert A.lib().dgx_attn_kv8_form(2, 3, 6, 8, 4, 128, 100, 0, 0, 0, None) == 1
    assert A.attn_kv8_form(0, 3, 6, 8, 4, 128, 100) == (0, 0, 0, 0)


def test_the_calls_of_the_gpu_tests_take_their_forms():
    """Every prompt tile, in one pass and in splits, and the split-KV form beside them."""
    seen = set()
    for heads, page, io, ctx, add, window, chunk, tile, split in [*G.CALLS.values(), *G.SMALL.values()]:
        f = G.form_of(heads, ctx, add, sum(add) + 3, window, chunk)
        assert f[0] == tile and (f[3] > 1) == split and f[1] in ((tile,) if tile else (16, 32, 64)), f
        seen.add((heads[2], f[0], f[3] > 1, window > 0))
    for HD, tiles in ((128, (64, 128)), (256, (64, 128)), (512, (64,))):
        for tile in tiles:
            for split in (False, True):
                assert (HD, tile, split, False) in seen and (HD, tile, split, True) in seen


def test_a_workspace_is_wanted_where_the_form_has_splits():
    for B in (1, 5, 16):
        for T in (1, 7, 40, 900):
            for NQ, NKV, HD in ((24, 4, 256), (16, 1, 512), (16, 8, 128)):
                for max_pos in (T, 500 + T, 20000):
                    for chunk in (0, 64, 1024):
                        for window in (0, 1, 300):
                            form = (ctypes.c_int * 4)()
                            assert A.lib().dgx_attn_kv8_form(B, T, B * T, NQ, NKV, HD, max_pos, chunk, window, 0, form) == 0
                            n = A.attn_kv8_workspace(B, T, B * T, NQ, NKV, HD, max_pos, chunk, window)
                            if form[3] > 1:
                                assert n >= B * T * NQ * form[3] * (HD + 2) * 4
                            elif T > 32:
                                assert n == 0


@pytest.mark.parametrize("window", [1, 2, 64, 1000, 4096])
def test_the_workspace_of_a_window_does_not_grow_with_the_positions(window):
    """Behind a window a row needs places for the splits of its request's keys alone: window + T - 1 neighbours."""
    for B, T, NQ, NKV, HD in ((16, 1, 16, 8, 256), (16, 8, 16, 8, 256), (64, 1, 24, 4, 256), (1, 500, 16, 8, 256), (3, 32, 16, 1, 512), (2, 3000, 8, 2, 128)):
        for chunk in (0, 64, 1024):
            for tree in (False, True)[:1 + (T <= 32)]:
                args = (B, T, B * T, NQ, NKV, HD)
                size = {A.attn_kv8_workspace(*args, mp, chunk, window, tree) for mp in (window + T + 40000, 131071, (1 << 30) - 1)}
                assert len(size) == 1
                C, ns = A.attn_kv8_form(*args, 131071, chunk, window, tree)[2:]
                if C:
                    lo = np.arange(min(C, 131072))                    # every place of the first key in its split
                    most = ((lo + window + T - 2) // C - lo // C + 1).max()
                    assert ns == min(131071 // C + 1, max(2, most)), (C, ns, most)
    assert A.attn_kv8_workspace(16, 8, 128, 16, 8, 256, 131071, window=1024) < 1 << 24


def test_the_device_check_without_the_raw_getter(monkeypatch):
    """A torch without the raw device getter: the checks ask torch.cuda, as the stream lookup does."""
    monkeypatch.setattr(A, "_get_device", None)
    monkeypatch.setattr(A.torch.cuda, "current_device", lambda: 1)
    A._here(1, "attn_kv8")
    for dev in (0, -1):
        with pytest.raises(ValueError):
            A._here(dev, "attn_kv8")


def test_a_bound_past_the_rows_is_the_rows():
    """T bounds a request's rows, which are no more than all rows: the form and the workspace are those of the smaller one."""
    for T in (6, 100, 1 << 26):
        for window, chunk in ((0, 0), (100, 64)):
            args = (2, 5, 24, 4, 256, 9000, chunk, window)
            assert A.attn_kv8_form(2, T, *args[1:]) == A.attn_kv8_form(2, 5, *args[1:])
            assert A.attn_kv8_workspace(2, T, *args[1:]) == A.attn_kv8_workspace(2, 5, *args[1:])
