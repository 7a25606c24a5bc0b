"""Refusals of the step over a paged cache and of the 4-bit pages, without a GPU: the C entry points check geometry and
pointers before they touch the device, and HipOps checks tensors before it takes their addresses."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from cellm_amd import _lib
from cellm_amd.hipops import HipOps

A = 1 << 20  # a 16-byte aligned address that no refused call reads
NAN, INF = float("nan"), float("inf")


@pytest.fixture()
def ctx():
    """Stands in for a context: every call here is refused before it looks into it."""
    buf = C.create_string_buffer(1 << 16)
    yield C.cast(buf, C.c_void_p)


def _calls():
    """name -> (arguments by name, in order)"""
    q4 = dict(kc=A, ks=A, vc=A, vs=A)
    head = dict(q=A, k=A, v=A, q_out=A, qw=A, kw=A, wdt=0, eps=1e-6, rows=4, nh=4, nkv=2, hd=64, pos=A, cs=A, positions=9,
                slots=A)
    tail = dict(total_blocks=8, n_layers=2, tpb=16, layer=1, stream=None)
    return {
        "kv_plan": dict(ctx=A, new=A, tables=3, bt=A, max_blocks=4, total_blocks=8, tpb=16, free=A, count=A, capacity=8, lens=A,
                        left=A, starts=A, pos=A, slots=A, rows=5, stream=None),
        "norm_rope_kv_write_f16": dict(**head, kc=A, vc=A, **tail),
        "norm_rope_kv_write_q8": dict(**head, **q4, **tail),
        "norm_rope_kv_write_q4": dict(**head, **q4, **tail),
        "kv_read_q4": dict(**q4, bt=A, max_blocks=4, total_blocks=8, pos=A, rows=4, per=2, nkv=2, hd=64, n_layers=2, tpb=16,
                           layer=1, dt=0, ko=A, vo=A, stream=None),
        "attention_gqa_q4kv": dict(q=A, **q4, bt=A, max_blocks=4, total_blocks=8, pos=A, rows=4, per=2, starts=None, tables=0,
                                   nh=4, nkv=2, hd=64, n_layers=2, tpb=16, layer=1, scale=0.0, cap=0.0, window=0, out=A,
                                   stream=None),
    }


BAD = [dict(hd=0), dict(hd=96), dict(hd=512), dict(nkv=0), dict(nkv=-1), dict(max_blocks=0), dict(max_blocks=1 << 31),
       dict(tpb=0), dict(max_blocks=1 << 62, tpb=4), dict(total_blocks=0), dict(total_blocks=-1), dict(total_blocks=1 << 33),
       dict(n_layers=0), dict(n_layers=1 << 40), dict(layer=2), dict(layer=-1), dict(rows=-1), dict(rows=3), dict(rows=1 << 21),
       dict(per=0), dict(per=-2), dict(nh=0), dict(nh=5), dict(nh=8192), dict(rows=1 << 20, nh=4096), dict(scale=-1.0),
       dict(scale=NAN), dict(scale=INF), dict(cap=-1.0), dict(cap=NAN), dict(cap=INF), dict(window=-1), dict(window=1 << 31),
       dict(positions=0), dict(dt=3), dict(dt=-1), dict(wdt=3), dict(wdt=-1), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF),
       dict(starts=A, tables=2, per=2), dict(starts=A, tables=-1, per=1), dict(starts=A, tables=(1 << 20) + 1, per=1),
       dict(tables=-1), dict(tables=(1 << 20) + 1), dict(capacity=-1), dict(capacity=1 << 31), dict(tpb=1 << 31),
       dict(max_blocks=(1 << 20) + 1, tpb=1), dict(max_blocks=1 << 16, tpb=1 << 15), dict(total_blocks=1 << 20, tpb=1 << 11),
       *[{p: None} for p in ("q", "k", "v", "q_out", "kc", "vc", "ks", "vs", "bt", "pos", "slots", "out", "ko", "vo", "ctx",
                             "new", "free", "count", "lens", "left", "starts")],
       *[{p: A + 8} for p in ("q", "k", "v", "q_out", "qw", "kw", "cs", "kc", "vc", "out", "ko", "vo")]]


def _applies(name, args, bad):
    if not all(p in args for p in bad):
        return False
    if name == "kv_plan":
        return "rows" not in bad or bad["rows"] != 3
    if "tables" in bad and "starts" not in bad or bad == dict(starts=None) or "capacity" in bad:
        return False  # without row_starts the number of tables is not looked at
    if bad == dict(total_blocks=1 << 20, tpb=1 << 11) or bad == dict(max_blocks=(1 << 20) + 1, tpb=1):
        return False  # the caches' own limits are wider
    if name.startswith("norm"):
        return bad not in (dict(rows=3), dict(nh=5), dict(rows=1 << 20, nh=4096))
    return True


@pytest.mark.parametrize("name", list(_calls()))
def test_bad_arguments_are_refused(ctx, name):
    fn = getattr(_lib.load(), "cellm_hip_" + name)
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


@pytest.mark.parametrize("name", ["norm_rope_kv_write_q4", "kv_read_q4", "attention_gqa_q4kv"])
def test_scales_of_four_bits_are_aligned(ctx, name):
    args = _calls()[name]
    for p in ("ks", "vs"):
        assert getattr(_lib.load(), "cellm_hip_" + name)(ctx, *{**args, p: A + 8}.values()) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("name", [n for n in _calls() if n != "kv_plan"])
def test_no_rows_is_no_work(ctx, name):
    args = _calls()[name]
    nulls = {p: None for p in args if args[p] == A}
    assert getattr(_lib.load(), "cellm_hip_" + name)(ctx, *{**args, **nulls, "rows": 0}.values()) == _lib.OK


def test_no_tables_is_no_attention(ctx):
    args = _calls()["attention_gqa_q4kv"]
    assert _lib.load().cellm_hip_attention_gqa_q4kv(ctx, *{**args, "starts": A, "per": 1}.values()) == _lib.OK


class _Unreachable:
    def __getattr__(self, name):
        return lambda *a: pytest.fail(f"{name} reached the C ABI with bad arguments")


class _OnDevice:
    """A host tensor that says it is on a device."""

    def __init__(self, t, device=0):
        self.t, self.d = t, device

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.d


@pytest.fixture()
def ops():
    o = HipOps.__new__(HipOps)
    o._lib, o._h, o.device = _Unreachable(), C.c_void_p(), 0
    return o


def _t(*shape, dtype=torch.float32):
    return _OnDevice(torch.zeros(*shape, dtype=dtype))


def _refused(call, args, changes):
    for name, bad in changes.items():
        with pytest.raises((TypeError, ValueError)):
            call(**{**args, **(bad if isinstance(bad, dict) else {name: bad})})


def test_plan_tensors(ops):
    i = torch.int32
    args = dict(context_lens_i32=_t(3, dtype=i), new_lens_i32=_t(3, dtype=i), block_tables=_t(3, 4, dtype=i), total_blocks=8,
                tokens_per_block=16, free_blocks=_t(8, dtype=i), free_count_i32=_t(1, dtype=i), lens_out=_t(3, dtype=i),
                free_out=_t(1, dtype=i), row_starts=_t(4, dtype=i), positions=_t(5, dtype=i), slots=_t(5, dtype=i))
    _refused(ops.encode_kv_plan, args, dict(
        context_lens_i32=_t(2, dtype=i), new_lens_i32=_t(3, dtype=torch.int64), block_tables=_t(12, dtype=i),
        free_blocks=torch.zeros(8, dtype=i), free_count_i32=_t(2, dtype=i), lens_out=_OnDevice(torch.zeros(3, dtype=i), 1),
        free_out=_t(1), row_starts=_t(3, dtype=i), positions=_OnDevice(torch.zeros(10, dtype=i)[::2]), slots=_t(4, dtype=i)))


def test_write_tensors(ops):
    i, u = torch.int32, torch.uint8
    args = dict(q=_t(5, 256), k=_t(5, 128), v=_t(5, 128), q_out=_t(5, 256), n_heads=4, n_kv_heads=2, head_dim=64,
                q_weight=_t(64), k_weight=_t(64), eps=1e-6, positions_i32=_t(5, dtype=i), cos_sin=_t(9, 32, 2),
                slots_i32=_t(5, dtype=i), kcache=_t(3, 1, 2, 4, 32, dtype=u), vcache=_t(3, 1, 2, 4, 32, dtype=u), total_blocks=3,
                n_layers=1, tokens_per_block=4, layer=0, kscale=_t(3, 1, 2, 4, 2, 2, dtype=torch.float16),
                vscale=_t(3, 1, 2, 4, 2, 2, dtype=torch.float16))
    _refused(ops.encode_norm_rope_kv_write, args, dict(
        q=_t(5, 255), k=_t(5, 128, dtype=torch.float16), v=_t(4, 128), q_out=torch.zeros(5, 256), q_weight=_t(63),
        k_weight=_t(64, dtype=torch.float16), positions_i32=_t(5, dtype=torch.int64), cos_sin=_t(9, 31, 2),
        slots_i32=_t(4, dtype=i), kcache=_t(3, 1, 2, 4, 64, dtype=u), vcache=_t(3, 1, 2, 4, 32, dtype=torch.int8),
        kscale=_t(3, 1, 2, 4, 2, 2), vscale=None, one=dict(kscale=None),
        eight=dict(kcache=_t(3, 1, 2, 4, 64, dtype=torch.int8), vcache=_t(3, 1, 2, 4, 64, dtype=torch.int8)),
        half=dict(kcache=_t(3, 1, 4, 2, 64, dtype=torch.float16), vcache=_t(3, 1, 4, 2, 64, dtype=torch.float16))))


def test_attention_and_read_tensors(ops):
    i, u, h = torch.int32, torch.uint8, torch.float16
    cache = dict(kcodes=_t(3, 1, 2, 4, 32, dtype=u), kscale=_t(3, 1, 2, 4, 2, 2, dtype=h), vcodes=_t(3, 1, 2, 4, 32, dtype=u),
                 vscale=_t(3, 1, 2, 4, 2, 2, dtype=h))
    geo = dict(n_kv_heads=2, head_dim=64, total_blocks=3, n_layers=1, tokens_per_block=4, layer=0)
    args = dict(q=_t(6, 256), **cache, block_tables=_t(6, 2, dtype=i), positions_i32=_t(6, dtype=i), out=_t(6, 256), n_heads=4,
                **geo)
    _refused(ops.encode_attention_q4, args, dict(
        q=_t(6, 255), kcodes=_t(3, 1, 2, 4, 32, dtype=torch.int8), kscale=_t(3, 1, 2, 4, 2, dtype=h), vcodes=_t(3, 1, 2, 4, 64, dtype=u),
        vscale=_t(3, 1, 2, 4, 2, 2), block_tables=_t(5, 2, dtype=i), positions_i32=_t(6), out=_t(6, 128), rows_per_table=4,
        starts=dict(row_starts_i32=_t(4, dtype=i)), both=dict(row_starts_i32=_t(7, dtype=i), rows_per_table=2),
        none=dict(row_starts_i32=_t(0, dtype=i)), wide=dict(row_starts_i32=_t(7, dtype=torch.int64))))
    args = dict(**cache, block_tables=_t(3, 2, dtype=i), positions_i32=_t(6, dtype=i), k_out=_t(6, 128), v_out=_t(6, 128),
                rows_per_table=2, **geo)
    _refused(ops.encode_kv_read_q4, args, dict(
        kcodes=_t(3, 1, 2, 4, 64, dtype=u), kscale=_t(3, 1, 2, 4, 2, 2), v_out=_t(6, 128, dtype=h), k_out=_t(6, 64),
        block_tables=_t(2, 2, dtype=i), rows_per_table=4,
        ints=dict(k_out=_t(6, 128, dtype=i), v_out=_t(6, 128, dtype=i))))
