"""The per-kernel times and callers built with an earlier header of the same
ABI: ``ai_attn_profile_read`` writes the kinds that ABI 9 began with, the others
are read with the size of the caller's arrays."""

import ctypes
import os
import re

import pytest

from conftest import ROOT
from autoindexer_b200 import _lib

GUARD = 12345


def _arrays(n, room):
    ms, cnt = (ctypes.c_float * room)(*[GUARD] * room), (ctypes.c_int32 * room)(*[GUARD] * room)
    return ms, cnt, lambda: (list(ms)[:n], list(cnt)[:n], list(ms)[n:] + list(cnt)[n:])


def test_read_fits_the_arrays_of_the_first_header():
    """Nine kinds: what a program built before the operators passes."""
    L = _lib.lib()
    assert L.ai_attn_abi_version() == 9
    ms, cnt, look = _arrays(9, 32)
    assert L.ai_attn_profile_enable(1) == 0
    assert L.ai_attn_profile_read(ms, cnt) == 0
    assert L.ai_attn_profile_enable(0) == 0
    a, b, rest = look()
    assert a == [0.0] * 9 and b == [0] * 9 and rest == [GUARD] * len(rest)


@pytest.mark.parametrize("room", [0, 1, 9, 13, 20])
def test_read_of_all_kinds_fits_the_room_it_is_given(room):
    L = _lib.lib()
    n = min(room, len(_lib.ALL_PROF_KINDS))
    ms, cnt, look = _arrays(n, 32)
    assert L.ai_attn_profile_enable(1) == 0
    assert L.ai_attn_profile_read_all(ms, cnt, room) == 0
    assert L.ai_attn_profile_enable(0) == 0
    a, b, rest = look()
    assert a == [0.0] * n and b == [0] * n and rest == [GUARD] * len(rest)


def test_refusals():
    L = _lib.lib()
    ms, cnt, _ = _arrays(9, 9)
    assert L.ai_attn_profile_read_all(None, cnt, 9) == 1
    assert L.ai_attn_profile_read_all(ms, None, 9) == 1
    assert L.ai_attn_profile_read_all(ms, cnt, -1) == 2


def test_header_lists_the_kinds():
    text = open(os.path.join(ROOT, "include", "ai_attn.h")).read()
    kinds = dict(re.findall(r"AI_PROF_(\w+) = (\d+)", text))
    assert int(kinds.pop("KINDS")) == len(_lib.PROF_KINDS) == 9
    assert int(kinds.pop("ALL_KINDS")) == len(_lib.ALL_PROF_KINDS)
    assert _lib.ALL_PROF_KINDS[:9] == _lib.PROF_KINDS
    assert [int(kinds[k.upper()]) for k in _lib.ALL_PROF_KINDS] == list(range(len(_lib.ALL_PROF_KINDS)))


@pytest.mark.gpu
def test_operators_are_timed(cuda_device):
    import torch

    from autoindexer_b200 import qk_norm_rope
    from autoindexer_b200.attention import KernelTimes

    q = torch.randn(1, 2, 3, 64, device=cuda_device)
    qk_norm_rope(q, q)
    with KernelTimes() as kt:
        qk_norm_rope(q, q)
    assert kt.launches["head_norm"] == 1 and kt.ms["head_norm"] > 0
    assert set(kt.launches) == set(_lib.ALL_PROF_KINDS) and sum(kt.launches.values()) == 1
