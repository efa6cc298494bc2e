"""The attention entry points' host code on the CPU (the HIP stand-in of tests/hoststub): what is refused, and with which
message; what reaches the kernels; nothing allocated, freed or set while a stream is captured."""
import ctypes as C
import importlib.util
from pathlib import Path

import numpy as np
import pytest

from ijah_amd.engine import AttnPromptC, Engine, EngineError, KvDesc, KvSeqs


@pytest.fixture(scope="module")
def host():
    spec = importlib.util.spec_from_file_location("hoststub_build_attn", Path(__file__).parent / "hoststub" / "build_attn.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    eng = Engine(mod.build())
    L = eng.lib
    L.hipstub_violations.restype, L.hipstub_violations.argtypes = C.c_int, [C.c_char_p, C.c_int]
    L.attnstub_scale.restype, L.attnstub_scale.argtypes = C.c_float, [C.c_int]
    L.attnstub_ld.restype, L.attnstub_ld.argtypes = C.c_long, [C.c_int]
    L.attnstub_base.restype = C.c_void_p
    return eng


@pytest.mark.parametrize("change,msg", [
    ({"dim": 96}, "dim 96"), ({"dim": 0}, "dim 0"), ({"dtype": 0}, "cache of type 0"), ({"dtype": 5}, "cache of type 5"),
    ({"pages": 0}, "0 pages"), ({"layers": -1}, "-1 layers"), ({"heads": 0}, "0 heads"), ({"pages": 2 ** 31 - 1}, "pages"),
    ({"pages": 2 ** 25 - 1, "heads": 65535, "layers": 65535}, "pages"), ({"heads": 65536}, "65536 heads")])
def test_create_refuses(host, change, msg):
    d = dict(layers=1, pages=4, heads=2, dim=64, dtype=2)
    d.update(change)
    assert host.lib.ne_kv_create(C.byref(KvDesc(**d))) is None
    assert msg in host.last_error(), host.last_error()
    assert host.lib.ne_kv_create(None) is None and "null" in host.last_error()


def test_info_and_null_handles(host):
    for dtype, e in (("BF16", 2), ("F16", 2), ("I8", 1)):
        kv = host.kv_create(3, 5, 2, 128, dtype)
        assert (kv.layers, kv.pages, kv.heads, kv.dim, kv.dtype) == (3, 5, 2, 128, dtype)
        assert kv.nbytes == 3 * 5 * 2 * (2 * 64 * 128 * e + (512 if e == 1 else 0))
    L = host.lib
    assert L.ne_kv_info(None, None, None) == -1
    assert L.ne_kv_write(None, 0, None, 1, None, 0, 0, None, 0, 0, 0, None) == -1 and "null cache" in host.last_error()
    assert L.ne_attn_decode(None, 0, None, 1, 1, None, 0, 0, None, 0, 0, 0, 1.0, None) == -1
    assert L.ne_attn_prompt(None, None) == -1 and "null" in host.last_error()
    L.ne_kv_free(None)
    assert L.attnstub_attrs() == 1  # at device set-up, once


class Calls:
    """a cache of 2 key heads of 64 and buffers for 3 rows of one sequence each"""

    def __init__(self, eng):
        self.eng, self.kv = eng, eng.kv_create(2, 4, 2, 64, "BF16")
        self.seqs = eng.kv_seqs(np.zeros((3, 2)), [1, 1, 1])
        self.k, self.v, self.q, self.out = (eng.alloc(3 * n * 64 * 4) for n in (2, 2, 4, 4))

    def write(self, seqs=None, layer=0, R=3, **kw):
        self.kv.write_bufs(layer, seqs or self.seqs, R, kw.pop("k", self.k), kw.pop("v", self.v), **kw)

    def attend(self, seqs=None, layer=0, R=3, heads=4, **kw):
        self.kv.attend_bufs(layer, seqs or self.seqs, R, heads, kw.pop("q", self.q), kw.pop("out", self.out), **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(layer=2), "layer 2"), (dict(layer=-1), "layer -1"), (dict(R=0), "rows 0"), (dict(R=2), "without `rows`"),
    (dict(R=2 ** 23), "rows 8388608"), (dict(ldk=100), "row stride 100"), (dict(ldv=129), "16-byte"),
    (dict(ldv=132), "too small"), (dict(k_off=8), "16-byte"), (dict(v_off=16), "v buffer too small"),
    (dict(k_off=2 ** 64 - 16), "k buffer too small"), (dict(dtype="I8"), "rows of type"), (dict(ldk=-128), "row stride -128")])
def test_write_refuses(host, kw, msg):
    c, before = Calls(host), host.lib.attnstub_launches()
    with pytest.raises(EngineError, match=msg):
        c.write(**kw)
    assert host.lib.attnstub_launches() == before


@pytest.mark.parametrize("kw,msg", [
    (dict(heads=3), "3 query heads over 2"), (dict(heads=0), "0 query heads"), (dict(heads=-2), "query heads"),
    (dict(heads=6), "q buffer too small"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=-1.0), "scale"), (dict(layer=5), "layer 5"), (dict(q_off=4), "16-byte"),
    (dict(ldo=255), "row stride 255")])
def test_decode_refuses(host, kw, msg):
    c, before = Calls(host), host.lib.attnstub_launches()
    with pytest.raises(EngineError, match=msg):
        c.attend(**kw)
    assert host.lib.attnstub_launches() == before


def test_sequences_refused(host):
    c, e = Calls(host), host
    small, ok = e.alloc(8), e.from_numpy(np.zeros(16, np.int32))
    for seqs, msg in ((KvSeqs(0, 1, ok, ok), "sequences 0"), (KvSeqs(3, 0, ok, ok), "table row length 0"),
                      (KvSeqs(3, 2 ** 30, ok, ok), "table row length"), (KvSeqs(3, 2, small, ok), "table buffer"),
                      (KvSeqs(3, 2, ok, small), "lens buffer"), (KvSeqs(3, 2, ok, ok, small), "rows buffer")):
        for call in (c.write, c.attend):
            with pytest.raises(EngineError, match=msg):
                call(seqs)
    null = KvSeqs(3, 2, ok, ok)
    null.c.table = None
    with pytest.raises(EngineError, match="null table"):
        c.write(null)
    assert e.lib.ne_kv_write(c.kv.ptr, 0, None, 1, c.k.ptr, 0, 0, c.v.ptr, 0, 0, 0, None) == -1
    assert "null sequences" in e.last_error()


def test_decode_in_place_or_apart(host):
    c = Calls(host)
    c.attend(out=c.q)  # its own rows
    wide = host.alloc(3 * 4 * 64 * 4 * 2)
    c.attend(q=wide, out=wide, ldq=512, ldo=512, out_off=0)
    c.attend(q=wide, out=wide, out_off=3 * 4 * 64 * 4)
    with pytest.raises(EngineError, match="overlaps q"):
        c.attend(q=wide, out=wide, out_off=16)
    with pytest.raises(EngineError, match="overlaps q"):
        c.attend(q=wide, out=wide, ldq=512)


PROMPT = dict(n=2, heads=4, kv_heads=2, dim=64, dtype=0, Rq=10, Rk=10, scale=0.125)


@pytest.mark.parametrize("change,msg", [
    (dict(dim=80), "dim 80"), (dict(heads=3), "3 query heads"), (dict(kv_heads=0), "over 0"), (dict(n=0), "sequences 0"),
    (dict(Rq=0), "rows 0"), (dict(Rk=11), "11 key rows"), (dict(dtype=8), "rows of type 8"), (dict(scale=0.0), "scale"),
    (dict(ldq=20), "row stride"), (dict(ldk=130), "16-byte"), (dict(ldv=132), "v buffer too small"), (dict(q_off=2), "16-byte"),
    (dict(q_rows=None), "null q_rows"), (dict(n=10), "q_rows buffer"), (dict(out="q"), "overlaps"), (dict(out="k"), "overlaps"),
    (dict(v=None), "null v"), (dict(Rq=2 ** 22, Rk=2 ** 22, heads=1024, kv_heads=1024), "rows of 2 sequences")])
def test_prompt_refuses(host, change, msg):
    e, before = host, host.lib.attnstub_launches()
    bufs = {"q": e.alloc(10 * 256 * 4), "k": e.alloc(10 * 256 * 4), "v": e.alloc(10 * 128 * 4), "out": e.alloc(10 * 256 * 4),
            "q_rows": e.from_numpy(np.array([0, 4, 10], np.int32))}
    fields = {**PROMPT, **{n: b.ptr for n, b in bufs.items()}}
    for n, v in change.items():
        fields[n] = bufs[v].ptr if isinstance(v, str) else v
    assert e.lib.ne_attn_prompt(C.byref(AttnPromptC(**fields)), None) == -1
    assert msg in e.last_error(), e.last_error()
    assert e.lib.attnstub_launches() == before
    fields.update({**PROMPT, "v": bufs["v"].ptr, "q_rows": bufs["q_rows"].ptr, "out": bufs["out"].ptr, "ldq": 0, "ldk": 0,
                   "ldv": 0, "q_off": 0})
    assert e.lib.ne_attn_prompt(C.byref(AttnPromptC(**fields)), None) == 0, e.last_error()
    assert abs(e.lib.attnstub_scale(1) - 0.125 * 1.4426950408889634) < 1e-7


def test_layers_strides_and_scale_reach_the_kernels(host):
    c = Calls(host)
    c.write(layer=0)
    base = host.lib.attnstub_base()
    c.write(layer=1)
    assert host.lib.attnstub_base() - base == 4 * 2 * 2 * 64 * 64 * 2
    assert host.lib.attnstub_ld(0) == 128
    wide = host.alloc(3 * 200 * 4)
    c.write(k=wide, ldk=200)
    assert host.lib.attnstub_ld(0) == 200 and host.lib.attnstub_ld(1) == 128
    c.attend()
    assert abs(host.lib.attnstub_scale(0) - 0.125 * 1.4426950408889634) < 1e-7


def test_calls_under_capture(host):
    """a captured step allocates, frees, sets and waits for nothing"""
    c = Calls(host)
    qr = host.from_numpy(np.array([0, 3], np.int32))
    host.lib.hipstub_reset()
    assert host.lib.hipstub_begin_capture() == 0
    c.write()
    c.kv.read_bufs(0, c.seqs, 3, c.k, c.v)
    c.attend()
    host.attn_prompt_bufs(1, qr, None, 3, 3, 4, 2, 64, c.q, c.k, c.v, c.out)
    assert host.lib.hipstub_end_capture() == 0
    buf = C.create_string_buffer(4096)
    assert host.lib.hipstub_violations(buf, 4096) == 0, buf.value.decode()


def test_read_refuses_pack_tensors(host, tmp_path):
    from ijah_amd import synth
    synth.write_safetensors(tmp_path / "m.safetensors", {"a": np.zeros((3, 128), np.float32)})
    p = host.pack_open(tmp_path)
    c = Calls(host)
    c.write(k=p.info("a").buf)
    with pytest.raises(EngineError, match="read-only"):
        c.kv.read_bufs(0, c.seqs, 3, p.info("a").buf, c.v)
