"""Clip-token operators without a GPU: the C entries' argument checks (nothing is launched, the pointers are never read), the refusal of
CPU tensors, and the row -> token arithmetic of packed query heads."""
import ctypes

import pytest
import torch

from slotvps_amd import _lib, ops

P = ctypes.c_void_p(4096)


def _ll(*v):
    return (ctypes.c_longlong * 3)(*v)


def test_attention_arguments():
    lib = _lib.load()
    s = _ll(64, 32, 16)

    def fwd(q=P, sq=s, out=P, ws=P, nb=1 << 40, B=1, N=4, M=4, H=2, Hk=2, D=16, frame=0, window=0, scale=0.25, dt=0):
        return lib.svps_attention_fwd(q, sq, P, s, P, s, out, None, None, None, ws, nb, B, N, M, H, Hk, D, frame, window, scale, dt, None)
    assert fwd(q=None) == -1 and fwd(sq=None) == -1 and fwd(out=ctypes.c_void_p(4104)) == -1 and fwd(sq=_ll(64, 33, 16)) == -1
    assert fwd(scale=0.0) == -1 and fwd(scale=float("nan")) == -1 and fwd(frame=-1) == -1 and fwd(window=1) == -1 and fwd(dt=2) == -1
    assert fwd(D=12) == -2 and fwd(D=136) == -2 and fwd(H=3) == -2 and fwd(B=0) == -2 and fwd(N=0) == -2 and fwd(M=0) == -2
    assert fwd(N=1 << 30, H=4) == -2 and fwd(B=1 << 20, N=1 << 20) == -2
    need = lib.svps_attention_workspace_bytes(1, 1, 1 << 20, 2, 2, 16)              # one query, a long memory: split over the keys
    assert need > 0 and fwd(N=1, M=1 << 20, nb=need - 1) == -3 and fwd(N=1, M=1 << 20, ws=None) == -3
    assert lib.svps_attention_workspace_bytes(0, 1, 1, 1, 1, 16) == 0 and lib.svps_attention_workspace_bytes(1, 1, 1, 3, 2, 16) == 0

    def bwd(lse=P, ws=P, nb=1 << 40, D=16, dt=0):
        return lib.svps_attention_bwd(P, s, P, s, P, s, P, s, P, lse, P, P, P, None, None, ws, nb, 1, 4, 4, 2, 2, D, 0, 0, 0.25, dt, None)
    assert bwd(lse=None) == -1 and bwd(ws=None) == -1 and bwd(dt=2) == -1 and bwd(D=20) == -2
    assert bwd(nb=lib.svps_attention_bwd_workspace_bytes(1, 4, 4, 2, 2, 16) - 1) == -3


def test_rotary_arguments():
    lib = _lib.load()
    turns = (ctypes.c_double * 128)()

    def rot(x=P, split=(4, 4), H=2, H2=0, D=16, ptype=0, pairing=0, dt=0, B=1, x2=None):
        c = (ctypes.c_int * len(split))(*split)
        return lib.svps_rotary_axes(x, _ll(32, 32, 16), P, H, x2, None, None, H2, P, 0, 1, ptype, len(split), c, turns, pairing, 0, dt, B, 3, D, None)
    assert rot(x=None) == -1 and rot(ptype=3) == -1 and rot(pairing=2) == -1 and rot(dt=3) == -1 and rot(H2=1) == -1
    assert rot(split=(3,)) == -2 and rot(split=(18,)) == -2 and rot(split=(2,) * 5) == -2 and rot(split=()) == -2 and rot(B=0) == -2
    assert rot(D=4097) == -2 and rot(D=600, split=(258,)) == -2 and rot(H=65536) == -2


def test_linear_arguments():
    lib = _lib.load()

    def fwd(x=P, act=0, dt=0, M=4, K=64, N=32, ldx=64, ws=None, nb=0):
        return lib.svps_linear_act_fwd(x, ldx, P, K, None, 0, None, act, P, None, ws, nb, M, K, N, dt, None)
    assert fwd(x=None) == -1 and fwd(act=3) == -1 and fwd(dt=2) == -1 and fwd(M=0) == -2 and fwd(ldx=63) == -2 and fwd(K=0) == -2
    assert fwd(K=63) == -3 and fwd(x=ctypes.c_void_p(4098)) == -3                   # operands that are copied need the workspace
    assert lib.svps_linear_act_workspace_bytes(4, 63, 32, 63, 63, 0) >= (4 + 32) * 64 * 2
    assert lib.svps_linear_act_workspace_bytes(4, 64, 32, 64, 64, 1) >= (4 + 32) * 64 * 2

    def bwd(dy=P, dx=P, dw=P, db=None, ldy=32, M=4, nb=1 << 40):
        return lib.svps_linear_act_bwd(dy, ldy, P, 64, P, 64, P, dx, dw, db, 0, P, nb, M, 64, 32, 0, None)
    assert bwd(dy=None) == -1 and bwd(dx=None, dw=None) == -1 and bwd(ldy=31) == -2 and bwd(M=0) == -2 and bwd(nb=0) == -3


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 4, 2, 16), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.rotary_axes(x, torch.zeros((4, 1), dtype=torch.int32), (4,))
    with pytest.raises(RuntimeError):
        ops.attention(x, x, x)
    with pytest.raises(RuntimeError):
        ops.linear_act(x, x[0, 0])


def test_division_by_the_group_size():
    """row // G as the kernels compute it: high word of row * (2^32 // G + 1), minus one where that is too far"""
    for G in (2, 3, 4, 5, 7, 8, 12, 24, 100, 1023, 65535):
        magic = (1 << 32) // G + 1
        rows = [r for b in (0, 1 << 10, 1 << 20, (1 << 30) + 128) for r in (b, b + 1, b + G - 1, b // G * G, b // G * G + G - 1, max(b // G * G - 1, 0))]
        for row in rows:
            n = row * magic >> 32
            n -= n * G > row
            assert n == row // G, (row, G)


def test_rotary_table():
    split, turns = ops._rotary_table((4, 8), 10000.0, "axis")
    assert list(split) == [4, 8] and len(turns) == 6
    two_pi = 6.283185307179586
    assert [round(t * two_pi, 12) for t in turns] == [1.0, 0.01, 1.0, 0.1, 0.01, 0.001]
    _, shared = ops._rotary_table((4, 8), 10000.0, "shared")
    assert abs(shared[5] * two_pi - 10000.0 ** (-10 / 12)) < 1e-15
