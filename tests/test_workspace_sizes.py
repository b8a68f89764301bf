"""Workspace sizes as a host uses them: taken once for its largest batch. None falls as an argument
rises."""

import pytest

import vastloom_b200 as vb

TOKENS = [0, 1, 2, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2048, 2049, 3000, 4095, 4096, 4097, 5000,
          8192, 8193, 12000, 16384, 16385, 32768, 32769, 65536, 1 << 20]
SEQS = [1, 2, 3, 4, 5, 7, 8, 9, 13, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 500, 4096]


@pytest.mark.parametrize("E", [1, 64, 256, 512])
def test_balance_workspace_never_falls(E):
    for S in SEQS:
        sizes = [vb.balance_workspace_bytes(T, E, S) for T in TOKENS]
        assert sizes == sorted(sizes), (S, sizes)
    for T in TOKENS:
        sizes = [vb.balance_workspace_bytes(T, E, S) for S in SEQS]
        assert sizes == sorted(sizes), (T, sizes)
        assert vb.balance_workspace_bytes(T, E, 13) <= vb.balance_workspace_bytes(T, E + 1, 13)


def test_int8_workspace_never_falls():
    rows, cols = [0, 1, 2, 7, 8, 24, 25, 100, 1000, 4095, 4096, 4097, 65536], [1, 15, 16, 17, 1000, 4096, 4097, 131071]
    for c in cols:
        sizes = [vb.int8_workspace_bytes(r, c) for r in rows]
        assert sizes == sorted(sizes), (c, sizes)
    for r in rows:
        sizes = [vb.int8_workspace_bytes(r, c) for c in cols]
        assert sizes == sorted(sizes), (r, sizes)


@pytest.mark.parametrize("k,E", [(1, 1), (8, 64), (6, 256), (8, 512)])
def test_route_plan_workspace_never_falls(k, E):
    lib = vb.load_library()
    sizes = [lib.vlb_ep_workspace_bytes(T, k, E) for T in TOKENS]
    assert sizes == sorted(sizes)
    assert lib.vlb_ep_workspace_bytes(1000, k, E) <= lib.vlb_ep_workspace_bytes(1000, k + 1, E + 1)
