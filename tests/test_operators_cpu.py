"""Refusals of the embedding, rotation, log-probability and AdamW operators before any launch, and the rotation's plan."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from memorax_b200.build import build_library
    build_library()
    from memorax_b200 import _lib
    return _lib.lib


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 4096)()
    yield (ctypes.addressof(buf) + 255) & ~255
    del buf


def test_embedding_validation(lib, p):
    def fwd(ids=p, width=8, table=p, out=p, keep=None, size=0, rows=4, vocab=9, dim=8, type=1):
        return lib.mxk_embedding_fwd(ids, width, table, out, keep, size, rows, vocab, dim, type, 1.0, None)
    assert fwd(ids=None) == fwd(table=None) == fwd(out=None) == -1
    assert fwd(rows=0) == fwd(vocab=0) == fwd(dim=0) == fwd(dim=2 ** 24 + 1) == fwd(rows=2 ** 31) == fwd(vocab=2 ** 31 - 1) == -2
    assert fwd(type=3) == fwd(width=2) == -4
    assert fwd(ids=p + 4) == fwd(table=p + 1) == fwd(out=p + 2, type=0) == fwd(keep=p + 8, size=1 << 20) == -3
    held = lib.mxk_embedding_sorted_bytes(100, 9)
    assert held == 2 * 1024 + 256 and lib.mxk_embedding_sorted_bytes(0, 9) == 0 and fwd(keep=p, size=held - 1, rows=100) == -5
    need = lib.mxk_embedding_bwd_workspace_bytes(100, 16)
    assert need == 4 * 2 * 16 * 4 and lib.mxk_embedding_bwd_workspace_bytes(0, 16) == 0
    def bwd(keep=p, kept=held, dy=p, dw=p, ws=p, size=1 << 20, rows=100, dim=16):
        return lib.mxk_embedding_bwd(keep, kept, dy, dw, ws, size, rows, 9, dim, 1, 1.0, None)
    assert bwd(keep=None) == bwd(dy=None) == bwd(dw=None) == -1 and bwd(rows=-1) == -2
    assert bwd(ws=None) == bwd(size=need - 1) == bwd(kept=held - 1) == -5 and bwd(ws=p + 8) == bwd(keep=p + 8) == -3


def test_logprob_validation(lib, p):
    def fwd(x=p, ld=40, tokens=p, width=8, lp=p, h=p, tv=p, ti=p, stats=p, rows=3, vocab=40, top=2, type=0, t=1.0):
        return lib.mxk_token_logprob_fwd(x, ld, None, 0, tokens, width, lp, h, tv, ti, stats, rows, vocab, top, type, t, None)
    assert fwd(x=None) == fwd(lp=None) == fwd(tv=None) == fwd(ti=None) == -1
    assert fwd(rows=0) == fwd(vocab=0) == fwd(top=41) == fwd(top=-1) == fwd(rows=2 ** 31) == fwd(vocab=2 ** 30) == -2
    assert fwd(type=5) == fwd(width=1) == fwd(top=33) == fwd(t=0.0) == fwd(t=-1.0) == fwd(t=math.nan) == fwd(t=math.inf) == -4
    assert fwd(x=p + 2) == fwd(tokens=p + 4) == fwd(stats=p + 4) == -3
    bwd = lambda stats=p, dx=p: lib.mxk_token_logprob_bwd(p, 40, None, 0, p, 8, stats, p, 1, p, 1, dx, 3, 40, 0, 1.0, None)
    assert bwd(stats=None) == bwd(dx=None) == -1 and bwd(stats=p + 4) == bwd(dx=p + 1) == -3


class Side(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("st", ctypes.c_longlong), ("sh", ctypes.c_longlong), ("dy", ctypes.c_void_p),
                ("db", ctypes.c_longlong), ("dt", ctypes.c_longlong), ("dh", ctypes.c_longlong), ("w", ctypes.c_void_p), ("out", ctypes.c_void_p), ("heads", ctypes.c_int)]


class Rotate(ctypes.Structure):
    _fields_ = [("side", Side * 2), ("positions", ctypes.c_void_p), ("positions_bytes", ctypes.c_int), ("pb", ctypes.c_longlong), ("pt", ctypes.c_longlong),
                ("turns", ctypes.c_void_p), ("batch", ctypes.c_longlong), ("steps", ctypes.c_longlong), ("dim", ctypes.c_int), ("rot", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("norm", ctypes.c_int), ("type", ctypes.c_int), ("eps", ctypes.c_float)]


def test_rotate_validation(lib, p):
    def args(**kw):
        side = lambda **s: Side(**{"x": p, "sb": 512, "st": 64, "sh": 32, "dy": p, "db": 512, "dt": 64, "dh": 32, "out": p, "heads": 2, **s})
        return Rotate(**{"side": (Side * 2)(side(**kw.pop("q", {})), side(**kw.pop("k", {}))), "turns": p, "batch": 2, "steps": 8, "dim": 32, "rot": 32, "norm": 1, "type": 1,
                         "eps": 1e-6, **kw})
    fwd = lambda **kw: lib.mxk_norm_rotate_fwd(ctypes.byref(args(**kw)), None)
    assert lib.mxk_norm_rotate_fwd(None, None) == fwd(turns=None) == fwd(q={"x": None}) == fwd(k={"out": None}) == -1
    assert fwd(batch=0) == fwd(steps=0) == fwd(dim=0) == fwd(dim=514) == fwd(rot=0) == fwd(rot=34) == fwd(q={"heads": 0}) == -2
    assert fwd(dim=31, rot=30) == fwd(rot=31) == fwd(type=7) == fwd(norm=3) == fwd(q={"w": p}) == fwd(norm=2, q={"w": p}, k={"w": p}) == -4
    assert fwd(positions=p, positions_bytes=2) == -4 and fwd(q={"x": p + 1}) == -3
    need = lib.mxk_norm_rotate_bwd_workspace_bytes(32)
    bwd = lambda ws=p, size=need, **kw: lib.mxk_norm_rotate_bwd(ctypes.byref(args(**kw)), p, p, ws, size, None)
    assert bwd(q={"dy": None}) == -1 and bwd(q={"w": p}, k={"w": p}, ws=None) == bwd(q={"w": p}, k={"w": p}, size=need - 1) == -5


class AdamTensor(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("g", ctypes.c_void_p), ("master", ctypes.c_void_p), ("n", ctypes.c_longlong), ("state", ctypes.c_longlong)]


class AdamState(ctypes.Structure):
    _fields_ = [("m", ctypes.c_void_p), ("v", ctypes.c_void_p), ("m_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("now", ctypes.c_void_p), ("bits", ctypes.c_int)]


def test_adamw_validation(lib, p):
    def step(count=1, types=(1, 1), number=1, tensors=True, state=True, t={}, s={}):
        one = (AdamTensor * 1)(AdamTensor(**{"p": p, "g": p, "master": None, "n": 8, "state": 0, **t}))
        st = AdamState(**{"m": p, "v": p, "m_scale": None, "v_scale": None, "now": None, "bits": 32, **s})
        return lib.mxk_adamw(one if tensors else None, count, *types, ctypes.byref(st) if state else None, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, number, None)
    assert step(tensors=False) == step(state=False) == step(t={"p": None}) == step(t={"g": None}) == step(s={"m": None}) == step(s={"bits": 8}) == -1
    assert step(count=0) == step(number=0) == step(t={"n": 0}) == step(t={"state": -256}) == -2
    assert step(types=(3, 3)) == step(types=(1, 2)) == step(types=(0, 1)) == step(s={"bits": 4}) == -4
    assert step(t={"p": p + 1}) == step(t={"state": 8}) == step(s={"m": p + 4}) == step(t={"master": p + 2}) == -3
    assert lib.mxk_adamw_tick(None, p, 0.9, 0.99, 0.0, p, None) == -1


def test_there_is_no_cpu_path():
    from memorax_b200 import blocks, ops
    plan = ops.RotaryPlan(8, device="cpu")
    for call in (lambda: ops.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(3, 4)), lambda: ops.token_log_probs(torch.zeros(3, 4)),
                 lambda: ops.norm_rotate(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8), plan), lambda: blocks.AdamW([torch.zeros(3)])):
        with pytest.raises(ValueError):
            call()


def test_rotary_plan():
    from memorax_b200 import ops
    plan = ops.RotaryPlan(128, base=500000.0, device="cpu")
    assert plan.turns.shape == (64,) and plan.turns.dtype == torch.int64
    for i, t in enumerate(plan.turns.tolist()):
        want = 500000.0 ** (-2 * i / 128) / (2 * math.pi)
        assert abs((t % 2 ** 64) / 2 ** 64 - want) <= 1e-15 * want + 2.0 ** -64
    given = ops.RotaryPlan(4, rates=[7.0, -0.5], device="cpu").turns.tolist()      # more than a turn, and backwards
    assert abs(given[0] % 2 ** 64 / 2 ** 64 - (7.0 / (2 * math.pi) - 1)) < 1e-15 and abs(given[1] / 2 ** 64 + 0.5 / (2 * math.pi)) < 1e-15
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=4, rates=[1.0]), dict(rotary_dim=4, base=0.0)):
        with pytest.raises(ValueError):
            ops.RotaryPlan(**bad, device="cpu")
    with pytest.raises(ValueError):
        ops.norm_rotate(None, None, plan, norm="batch")
