"""Refusals of the paged 8-bit cache and drafted-tree calls, without a GPU: the C entry points
check geometry and pointers before they touch the device, and HipOps checks tensors before it
takes their addresses."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from cellm_amd import _lib
from cellm_amd.hipops import HipOps

A = 1 << 20  # a 16-byte aligned address that no refused call reads


@pytest.fixture()
def ctx():
    """Stands in for a context: every call here is refused before it looks into it."""
    buf = C.create_string_buffer(1 << 16)
    yield C.cast(buf, C.c_void_p)


def _calls():
    """name -> (arguments by name, in order)"""
    geo = dict(max_blocks=4, total_blocks=8, n_layers=2, tpb=16, layer=1)
    q8 = dict(kc=A, ks=A, vc=A, vs=A)
    return {
        "kv_write_q8": dict(k=A, v=A, rows=4, per=2, nkv=2, hd=64, pos=A, **q8, bt=A, **geo, stream=None),
        "rope_kv_write_q8": dict(q=A, k=A, v=A, q_out=A, rows=4, per=2, nh=4, nkv=2, hd=64, pos=A, slots=None, cs=A,
                                 positions=9, **q8, bt=A, **geo, stream=None),
        "kv_read_q8": dict(**q8, bt=A, max_blocks=4, total_blocks=8, pos=A, rows=4, per=2, nkv=2, hd=64, n_layers=2, tpb=16,
                           layer=1, dt=0, ko=A, vo=A, stream=None),
        "attention_gqa_q8kv": dict(q=A, **q8, bt=A, max_blocks=4, total_blocks=8, pos=A, rows=4, per=2, nh=4, nkv=2, hd=64,
                                   n_layers=2, tpb=16, layer=1, scale=0.0, cap=0.0, window=0, out=A, stream=None),
        "attention_tree_q8kv": dict(q=A, **q8, bt=A, max_blocks=4, total_blocks=8, pos=A, masks=A, tables=2, tree=5, nh=4,
                                    nkv=2, hd=64, n_layers=2, tpb=16, layer=1, scale=0.0, cap=0.0, window=0, out=A,
                                    stream=None),
        "attention_tree_f16kv": dict(q=A, kc=A, vc=A, bt=A, max_blocks=4, total_blocks=8, pos=A, masks=A, tables=2, tree=5,
                                     nh=4, nkv=2, hd=64, n_layers=2, tpb=16, layer=1, scale=0.0, cap=0.0, window=0, out=A,
                                     stream=None),
        "kv_accept_q8": dict(**q8, bt=A, max_blocks=4, total_blocks=8, pos=A, acc=A, most=3, tables=2, tree=5, nkv=2, hd=64,
                             n_layers=2, tpb=16, stream=None),
        "kv_accept_f16": dict(kc=A, vc=A, bt=A, max_blocks=4, total_blocks=8, pos=A, acc=A, most=3, tables=2, tree=5, nkv=2,
                              hd=64, n_layers=2, tpb=16, stream=None),
    }


NAN, INF = float("nan"), float("inf")
BAD = [dict(hd=0), dict(hd=96), dict(hd=512), dict(nkv=0), dict(nkv=-1), dict(max_blocks=0), dict(max_blocks=1 << 31),
       dict(tpb=0), dict(tpb=1 << 29), dict(max_blocks=1 << 62, tpb=4), dict(total_blocks=0), dict(total_blocks=-1),
       dict(total_blocks=1 << 33), dict(n_layers=0), dict(n_layers=1 << 40), dict(layer=2), dict(layer=-1), dict(rows=-1),
       dict(rows=3), dict(rows=1 << 21), dict(per=0), dict(per=-2), dict(total_blocks=1 << 28, tpb=16, nkv=2, n_layers=2),
       dict(nh=0), dict(nh=5), dict(nh=8192), dict(rows=1 << 20, nh=4096), dict(scale=-1.0), dict(scale=NAN),
       dict(scale=INF), dict(cap=-1.0), dict(cap=NAN), dict(cap=INF), dict(window=-1), dict(window=1 << 31), dict(window=4),
       dict(tree=0), dict(tree=257), dict(tables=-1), dict(tables=1 << 21), dict(most=0), dict(most=6), dict(positions=0),
       dict(dt=3), dict(dt=-1),
       *[{p: v} for p in ("q", "k", "v", "q_out", "cs", "kc", "vc", "ks", "vs", "bt", "pos", "masks", "out", "ko", "vo",
                          "acc") for v in ([None] if p in ("ks", "vs", "bt", "pos", "masks", "acc") else [None, A + 8])]]


def _applies(name, args, bad):
    if not all(p in args for p in bad):
        return False
    if "window" in bad and bad["window"] == 4:
        return "tree" in args
    if name.startswith(("kv_write", "rope")) and bad.get("nh") == 5:
        return False  # query heads are only turned: any number
    if name.startswith("rope") and bad == dict(rows=1 << 20, nh=4096):
        return False
    return True


@pytest.mark.parametrize("name", list(_calls()))
def test_bad_arguments_are_refused(ctx, name):
    lib = _lib.load()
    fn = getattr(lib, "cellm_hip_" + name)
    args = _calls()[name]
    seen = 0
    for bad in BAD:
        if not _applies(name, args, bad):
            continue
        rc = fn(ctx, *{**args, **bad}.values())
        assert rc in (_lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED), (name, bad, rc)
        assert _lib.last_error(), (name, bad)
        seen += 1
    assert seen > 15
    assert fn(None, *args.values()) == _lib.ERR_INVALID_ARG and "null context" in _lib.last_error()


@pytest.mark.parametrize("name", list(_calls()))
def test_no_rows_is_no_work(ctx, name):
    args = _calls()[name]
    none = dict(rows=0) if "rows" in args else dict(tables=0)
    nulls = {p: None for p in args if args[p] == A}
    assert getattr(_lib.load(), "cellm_hip_" + name)(ctx, *{**args, **nulls, **none}.values()) == _lib.OK


class _Unreachable:
    def __getattr__(self, name):
        return lambda *a: pytest.fail(f"{name} reached the C ABI with bad arguments")


class _OnDevice:
    """A host tensor that says it is on device 0."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 0


@pytest.fixture()
def ops():
    o = HipOps.__new__(HipOps)
    o._lib, o._h, o.device = _Unreachable(), C.c_void_p(), 0
    return o


def _tensors(**kw):
    z = dict(q=torch.zeros(4, 128), k=torch.zeros(4, 128), v=torch.zeros(4, 128), out=torch.zeros(4, 128),
             pos=torch.zeros(4, dtype=torch.int32), cs=torch.zeros(9, 32, 2), kc=torch.zeros(3, 1, 2, 16, 64, dtype=torch.int8),
             ks=torch.zeros(3, 1, 2, 16), vc=torch.zeros(3, 1, 2, 16, 64, dtype=torch.int8), vs=torch.zeros(3, 1, 2, 16),
             bt=torch.zeros(4, 2, dtype=torch.int32), ctx=torch.zeros(4, dtype=torch.int32),
             masks=torch.zeros(4, 1, 1, dtype=torch.int64), acc=torch.zeros(4, 1, dtype=torch.int32))
    z.update(kw)
    return {n: None if t is None else _OnDevice(t) if isinstance(t, torch.Tensor) else t for n, t in z.items()}


def _do(ops, what, t, per=1):
    geo, cache = (3, 1, 16, 0), (t["kc"], t["ks"], t["vc"], t["vs"])
    if what == "write":
        ops.encode_kv_write_q8(t["k"], t["v"], 2, 64, t["pos"], *cache, t["bt"], *geo, rows_per_table=per)
    elif what == "rope":
        ops.encode_rope_kv_write_q8(t["q"], t["k"], t["v"], t["out"], 2, 2, 64, t["pos"], t["cs"], *cache, t["bt"], *geo,
                                    slots_i32=t.get("slots"), rows_per_table=per)
    elif what == "read":
        ops.encode_kv_read_q8(*cache, t["bt"], t["pos"], t["k"], t["v"], 2, 64, *geo, rows_per_table=per)
    elif what == "attend":
        ops.encode_attention_q8(t["q"], *cache, t["bt"], t["pos"], t["out"], 2, 2, 64, *geo, rows_per_table=per)
    elif what == "tree":
        ops.encode_attention_tree(t["q"], t["kc"], t["vc"], t["bt"], t["ctx"], t["masks"], t["out"], 2, 2, 64, *geo,
                                  kscale=t["ks"], vscale=t["vs"])
    else:
        ops.encode_kv_accept(t["kc"], t["vc"], t["bt"], t["ctx"], t["acc"], 5, 2, 64, 3, 1, 16, kscale=t["ks"],
                             vscale=t["vs"])


I32, F16 = torch.int32, torch.float16
CASES = [
    ("write", dict(k=torch.zeros(3, 128))), ("write", dict(v=torch.zeros(4, 128, dtype=F16))),
    ("write", dict(pos=torch.zeros(4))), ("write", dict(kc=torch.zeros(2, 1, 2, 16, 64, dtype=torch.int8))),
    ("write", dict(ks=torch.zeros(3, 1, 2, 16, dtype=F16))), ("write", dict(bt=torch.zeros(3, 2, dtype=I32))),
    ("write", dict(bt=torch.zeros(4, 2, dtype=torch.int64))), ("rope", dict(q=torch.zeros(4, 64))),
    ("rope", dict(out=torch.zeros(4, 127))), ("rope", dict(cs=torch.zeros(9, 16, 2))),
    ("rope", dict(slots=torch.zeros(3, dtype=I32))), ("rope", dict(vs=torch.zeros(3, 1, 2, 15))),
    ("read", dict(k=torch.zeros(4, 128, dtype=F16))), ("read", dict(k=torch.zeros(4, 128, dtype=torch.float64))),
    ("read", dict(pos=torch.zeros(5, dtype=I32))), ("attend", dict(q=torch.zeros(4, 128).half())),
    ("attend", dict(out=torch.zeros(2, 128))), ("attend", dict(q=torch.zeros(128, 4).T)),
    ("attend", dict(kc=torch.zeros(3, 1, 2, 16, 64))), ("tree", dict(masks=torch.zeros(4, 1, dtype=torch.int64))),
    ("tree", dict(masks=torch.zeros(4, 1, 2, dtype=torch.int64))), ("tree", dict(masks=torch.zeros(4, 1, 1, dtype=I32))),
    ("tree", dict(ks=None)), ("tree", dict(ks=None, vs=None)), ("tree", dict(ctx=torch.zeros(2, dtype=I32))),
    ("accept", dict(acc=torch.zeros(4, dtype=I32))), ("accept", dict(acc=torch.zeros(3, 1, dtype=I32))),
    ("accept", dict(vs=None)), ("accept", dict(kc=torch.zeros(3, 1, 2, 16, 64, dtype=F16)))]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_bad_tensors_are_refused(ops, i):
    what, bad = CASES[i]
    with pytest.raises((ValueError, TypeError)):
        _do(ops, what, _tensors(**bad))


@pytest.mark.parametrize("what", ["write", "rope", "read", "attend", "tree", "accept"])
def test_host_tensors_and_rows_of_no_table_are_refused(ops, what):
    with pytest.raises(ValueError, match="device tensors"):
        _do(ops, what, {n: t.t for n, t in _tensors().items()})
    if what in ("write", "rope", "read", "attend"):
        for per in (0, 3, -1):
            with pytest.raises(ValueError, match="rows_per_table"):
                _do(ops, what, _tensors(), per)


@pytest.mark.parametrize("bad", [dict(rows=1 << 20, nh=4096), dict(rows=1 << 20, nh=510, hd=128),
                                 dict(rows=1 << 20, nh=63, hd=256)])
def test_more_threads_than_a_grid_numbers_are_refused(ctx, bad):
    args = _calls()["rope_kv_write_q8"]
    assert _lib.load().cellm_hip_rope_kv_write_q8(ctx, *{**args, **bad}.values()) == _lib.ERR_INVALID_ARG
    assert "2^34" in _lib.last_error()
