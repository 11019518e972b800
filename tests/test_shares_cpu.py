"""How paged_attention's work is shared out (csrc/shares.h), compiled for the host: the shares cover the work, and the join
follows no entry that would lead it out of its workspace."""

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "torch-xdna_b200" / "csrc"
SOURCE = """
#include "shares.h"
extern "C" long long begin_of(long long work, unsigned shares, long long i) { return xdna::Shares(work, shares).begin(i); }
extern "C" int owner_of(long long work, unsigned shares, long long unit) { return xdna::Shares(work, shares).owner(unit); }
extern "C" int exist(int first, int last, int slot, int shares) { return xdna::parts_exist(first, last, slot, shares); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    at = tmp_path_factory.mktemp("shares")
    (at / "shares.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(at / "shares.so"),
                    str(at / "shares.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "shares.so"))
    lib.begin_of.restype = ctypes.c_longlong
    lib.begin_of.argtypes = [ctypes.c_longlong, ctypes.c_uint, ctypes.c_longlong]
    lib.owner_of.argtypes = [ctypes.c_longlong, ctypes.c_uint, ctypes.c_longlong]
    return lib


@pytest.mark.parametrize("work", [0, 1, 7, 443, 444, 445, 10 ** 5, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 5])
@pytest.mark.parametrize("shares", [1, 3, 444, 1776])
def test_shares_cover_the_work(lib, work, shares):
    assert lib.begin_of(work, shares, 0) == 0 and lib.begin_of(work, shares, shares) == work
    g = random.Random(work + shares)
    for unit in {0, work // 2, work - 1} | {g.randrange(work) for _ in range(50)} if work else ():
        i = lib.owner_of(work, shares, unit)
        assert 0 <= i < shares and lib.begin_of(work, shares, i) <= unit < lib.begin_of(work, shares, i + 1)


def test_the_join_follows_what_the_kernel_writes(lib):
    """Of every item that begins inside a share: first share, the last unit's owner, slot 2 i or 2 i + 1."""
    g = random.Random(1)
    for _ in range(200):
        shares, items = g.choice([1, 5, 444, 1776]), [g.randrange(1, 60) for _ in range(g.randrange(1, 80))]
        work, at = sum(items), 0
        for n in items:
            first, last = lib.owner_of(work, shares, at), lib.owner_of(work, shares, at + n - 1)
            slot = 2 * first + (0 if at == lib.begin_of(work, shares, first) else 1)
            assert lib.exist(first, last, slot, shares)
            at += n


def test_the_join_follows_nothing_else(lib):
    """Entries that were not written hold anything: numbers of all sizes and signs, floats, codes, an earlier call's entries
    of more shares. What the join follows leads it to at most `shares` parts, all of them inside the workspace."""
    g = random.Random(2)
    odd = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 0x7f7f7f7f, -0x7f7f7f80, 0x3f800000, 0x7fc00000 - 2 ** 32, 443, 444, 888, 1775, 3551]
    for _ in range(20000):
        shares = g.choice([1, 2, 444, 1776])
        first, last, slot = (g.choice(odd) if g.random() < 0.5 else g.randrange(-4, 2 * shares + 4) for _ in range(3))
        if lib.exist(first, last, slot, shares):
            assert 0 <= first <= last < shares and 0 <= slot < 2 * shares
    assert not lib.exist(0, 2 ** 31 - 1, 0, 1776)        # would run on for billions of parts
    assert not lib.exist(-5, 3, -10, 1776) and not lib.exist(2, 1, 4, 1776) and not lib.exist(3, 5, 2 ** 30, 1776)
