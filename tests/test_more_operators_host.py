"""CPU: what the C entries of the mixture-of-experts step, the norms between blocks and the log-probabilities refuse, before
any launch."""

import ctypes

from xanosmerks_b200 import _lib

L, BAD, NO = _lib.lib, _lib.XM_ERR_INVALID, _lib.XM_ERR_UNSUPPORTED


def step(T=1, H=512, F=512, E=4, k=2, qtype=12, act=0, xs=None, rs=0, os=None, x=256, ws=256, n=1 << 40, dt=0, gate=256, w=256):
    return L.xm_moe_step(x, dt, T, H, H if xs is None else xs, None, 1e-5, gate, E, k, F, w, qtype, act, None, rs, 256,
                         H if os is None else os, ws, n, None)


def test_moe_step():
    assert step(T=0) == 0
    assert step(T=65) == BAD and step(T=-1) == BAD
    assert step(H=384) == NO and step(F=128) == NO and step(H=16640) == NO and step(H=0) == NO
    assert step(E=257) == NO and step(k=5) == NO and step(E=64, k=17) == NO and step(k=0) == NO
    assert step(qtype=0) == NO and step(qtype=16) == NO and step(act=4) == BAD and step(dt=3) == BAD
    assert step(xs=511) == BAD and step(os=511) == BAD
    assert step(x=None) == BAD and step(x=258) == BAD and step(ws=128) == BAD and step(gate=260) == BAD and step(w=32) == BAD
    need = L.xm_moe_step_workspace_size(1, 512, 512, 4, 2, 12)
    assert need > 0 and step(n=need - 1) == BAD and b"workspace" in L.xm_last_error()
    assert L.xm_moe_step_workspace_size(65, 512, 512, 4, 2, 12) == 0
    assert L.xm_moe_step_workspace_size(1, 500, 512, 4, 2, 12) == 0


def test_moe_step_table():
    E = 2
    assert L.xm_moe_step_table_size(0) == 0 and L.xm_moe_step_table_size(257) == 0
    host = ctypes.create_string_buffer(L.xm_moe_step_table_size(E))
    good, odd = (ctypes.c_void_p * E)(256, 512), (ctypes.c_void_p * E)(256, 520)

    def table(qtype=14, H=768, F=768, w1=good, w3=good, w2=good, to=host):
        return L.xm_moe_step_table(qtype, H, F, E, w1, w3, w2, to)

    assert table() == 0                                # (rows of 630 bytes: no tensor maps, the addresses alone)
    assert list((ctypes.c_uint64 * (3 * E)).from_buffer_copy(host.raw[-24 * E:])) == [256, 512] * 3
    assert table(w3=odd) == BAD and b"expert 1" in L.xm_last_error() and table(w1=None) == BAD and table(to=None) == BAD
    assert table(qtype=1) == NO and table(H=700) == NO


def norm(rows=1, D=64, ht=0, yt=0, hp=64, yp=64, op=64, gate=None, gt=0, gp=0, per=1, pre=None, nt=0, np_=64, h=256, nxt=None):
    return L.xm_residual_norm(h, ht, hp, 256, yt, yp, rows, D, None, gate, gt, gp, 0, per, 1.0, pre, 1e-5, 256, op, nxt, nt,
                              np_, None)


def test_residual_norm():
    assert norm(rows=0) == 0
    assert norm(rows=-1) == BAD and norm(D=0) == BAD and norm(D=32769, hp=40000, yp=40000, op=40000) == BAD
    assert norm(ht=3) == BAD and norm(yt=-1) == BAD and norm(gate=256, gt=9) == BAD and norm(pre=256, nt=5, nxt=256) == BAD
    assert norm(hp=63) == BAD and norm(yp=63) == BAD and norm(op=63) == BAD and norm(pre=256, nxt=256, np_=63) == BAD
    assert norm(gate=256, per=0) == BAD and norm(h=None) == BAD and norm(pre=256) == BAD and norm(h=257) == BAD


def logp(B=1, V=100, dt=0, stride=100, tb=8, top=0, x=256, tok=256, ids=256):
    return L.xm_logprobs(x, dt, B, V, stride, tok, tb, 1.0, None, top, 256, 256, 256, ids, 256, None)


def test_logprobs():
    assert logp(B=0) == 0
    assert logp(dt=4) == BAD and logp(V=0) == BAD and logp(V=(1 << 20) + 1, stride=1 << 21) == BAD and logp(stride=99) == BAD
    assert logp(tb=2) == BAD and logp(top=65) == BAD and logp(top=101) == BAD and logp(top=-1) == BAD and logp(B=-1) == BAD
    assert logp(x=None) == BAD and logp(x=258) == BAD and logp(tok=260) == BAD and logp(top=1, ids=None) == BAD
