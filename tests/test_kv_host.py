"""The paged cache's operators and beam search (include/gsk.h) without a GPU: the oracle's pins, the binding's structs against the
header, and the refusals of the Python layer."""
import ctypes as C
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import kv_ref as kr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, HF, F32, E4, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


# ---- the oracle ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [E4, I8])
def test_8_bits_are_the_nearest_value(dtype):
    """Against a search over every value that 8 bits hold; of two at one distance, the one with an even last bit."""
    held = torch.arange(256, dtype=torch.uint8).view(dtype).float().double().numpy()
    held = held[np.isfinite(held)]
    rng = np.random.default_rng(0)
    x = rng.normal(size=(50, 16)) * np.exp(3 * rng.normal(size=(50, 1)))
    x[0], x[1, 1:] = 0, 0
    y, s = kr.to_8(x, dtype)
    for row, got, scale in zip(x, y, s):
        assert scale == max(np.float32(np.abs(row).max()) * np.float32(1 / kr.MOST[dtype]), np.float32(2 ** -126))
        z = (row * float(np.float32(1) / scale)).astype(np.float32).astype(np.float64)
        near = np.abs(held[None] - z[:, None]).min(1)
        assert (np.abs(got - z) == near).all() and np.isin(got, held).all()
    tie = np.array([[kr.MOST[dtype]] + [k + 0.5 for k in range(15)]])
    assert kr.to_8(tie, dtype)[1][0] in (1.0, np.nextafter(np.float32(1), np.float32(2)), np.nextafter(np.float32(1), np.float32(0)))
    bad, s = kr.to_8(np.array([[1, np.nan], [np.inf, 2], [1, 2]]), dtype)
    assert np.isnan(s[:2]).all() and (bad[:2] == 0).all() and s[2] > 0


def test_attend_closed_forms():
    """Equal scores: the mean; one score far above: its value; a mask's row that sees nothing: 0; NaN where nothing looks."""
    k, v = np.zeros((6, 2, 8)), np.arange(96.0).reshape(6, 2, 8)
    q = np.ones((3, 4, 8))
    mask = np.zeros((3, 6), bool)
    mask[0, :4], mask[1, 2] = True, True
    v[5] = np.nan
    out, tol = kr.attend(q, k, v, mask, 0.5, BF, False)
    assert np.allclose(out[0, 0], v[:4, 0].mean(0)) and np.allclose(out[0, 3], v[:4, 1].mean(0))
    assert np.allclose(out[1, 1], v[2, 0]) and (out[2] == 0).all() and (tol[2] == 0).all() and (tol[0] > 0).all()
    k[3, 0] = 100
    assert np.allclose(kr.attend(q, k, v, mask, 0.5, BF, False)[0][0, 1], v[3, 0])


def test_what_a_node_sees():
    m = kr.sees(5, 2, parents=[9, 9, -1, 2, 2, 3, 77], begin=2)
    assert m.astype(int).tolist() == [[1, 1, 1, 0, 0, 0, 0], [1, 1, 1, 1, 0, 0, 0], [1, 1, 1, 0, 1, 0, 0], [1, 1, 1, 1, 0, 1, 0],
                                      [1, 1, 0, 0, 0, 0, 1]]
    assert kr.sees(3, 1).astype(int).tolist() == [[1, 1, 0, 0], [1, 1, 1, 0], [1, 1, 1, 1]]


def test_beams_known_answer():
    x = np.log(np.array([[0.5, 0.25, 0.25, 0.0 + 1e-300], [0.5, 0.5, 1e-300, 1e-300]]))
    x[0, 3] = x[1, 2] = x[1, 3] = -np.inf
    got = kr.beams(x, [0.0, math.log(0.5)], 9)
    assert [(t, b) for t, b, _ in got] == [(0, 0), (1, 0), (2, 0), (0, 1), (1, 1)]
    assert np.allclose([s for _, _, s in got], np.log([0.5, 0.25, 0.25, 0.25, 0.25]))


# ---- the binding -----------------------------------------------------------------------------------------------------

def test_structs_and_symbols_match_the_header(ge, tmp_path):
    lib = ge._lib
    header = os.path.join(ROOT, "include", "gsk.h")
    names = set(re.findall(r"GSE_API\s+[\w\s\*]+?\b(gsk_\w+)\s*\(", open(header).read()))
    assert names == set(lib.KV_SIGNATURES)
    L = lib.bind()
    pairs = [("gsk_cache", lib.KvCache), ("gsk_rows", lib.KvRows), ("gsk_read_rows", lib.KvRead), ("gsk_attention", lib.Attention),
             ("gsk_beams", lib.Beams), ("gsk_reorder_beams", lib.Reorder)]
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "gsk.h"\nint main(void) {\n'
    for t, cls in pairs:
        src += f'printf("%zu\\n", sizeof({t}));\n' + "".join(f'printf("%zu\\n", offsetof({t}, {f}));\n' for f, _ in cls._fields_)
    consts = ["GSK_BF16", "GSK_F16", "GSK_F32", "GSK_E4M3", "GSK_I8", "GSK_MAX_DIM", "GSK_MAX_TREE", "GSK_MAX_BEAMS", "GSK_MAX_KEEP"]
    src += "".join(f'printf("%d\\n", {c});\n' for c in consts) + "}\n"
    (tmp_path / "a.c").write_text(src)
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")],
                   check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want + [lib.K_BF16, lib.K_F16, lib.K_F32, lib.K_E4M3, lib.K_I8, lib.MAX_DIM, lib.MAX_TREE, lib.MAX_BEAMS, lib.MAX_KEEP]
    for n in names:  # no handle, no call
        assert getattr(L, n)(*([None] * len(lib.KV_SIGNATURES[n][1]))) == lib.E_ARG


# ---- refusals --------------------------------------------------------------------------------------------------------

def _refusals(call, ok, bad):
    for kw in bad:
        with pytest.raises(ValueError):
            call(**{**ok, **kw})
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="HIP device"):
            call(**ok)


def _caches(dtype=BF, shape=(6, 4, 3, 16)):
    return torch.zeros(shape).to(dtype), torch.zeros(shape).to(dtype)


def _scales(shape=(6, 4, 3)):
    return torch.zeros(shape), torch.zeros(shape)


def _bad_caches():
    k, v = _caches()
    k8, v8 = _caches(E4)
    wide = torch.zeros(6, 4, 3, 19, dtype=BF)
    return [dict(keys=k.float(), values=v.float()), dict(values=v[:5]), dict(values=v.half()), dict(keys=k[0], values=v[0]),
            dict(values=v.transpose(1, 2).contiguous().transpose(1, 2)), dict(keys=wide[..., :16], values=wide[..., :16]),
            dict(keys=wide[..., 1:17], values=wide[..., 1:17]), dict(keys=wide[..., :12].contiguous(), values=wide[..., :12].contiguous()),
            dict(keys=k.repeat(1, 1, 1, 17), values=v.repeat(1, 1, 1, 17)), dict(keys=k[:0], values=v[:0]),
            dict(keys=k.transpose(2, 3), values=v.transpose(2, 3)), dict(scales=_scales()),
            dict(keys=k8, values=v8), dict(keys=k8, values=v8, scales=(_scales()[0], _scales()[1][:5])),
            dict(keys=k8, values=v8, scales=tuple(s.half() for s in _scales())),
            dict(keys=k8, values=v8, scales=(_scales()[0], torch.zeros(6, 3, 4).transpose(1, 2)))]


def test_write_refuses(ge):
    k, v = _caches()
    x = torch.zeros(5, 3, 16, dtype=BF)
    ok = dict(slot=torch.zeros(5, dtype=torch.int64), k=x, v=x, keys=k, values=v)
    k8, _ = _caches(I8)
    s = _scales()[0]
    _refusals(ge.kv.write, ok, [*_bad_caches(), dict(values=k), dict(keys=k[:1].expand(6, 4, 3, 16), values=v[:1].expand(6, 4, 3, 16)),
                                dict(slot=ok["slot"].int()), dict(slot=ok["slot"][:4]), dict(slot=ok["slot"][None]), dict(k=x[:4]),
                                dict(k=x[:, :2]), dict(k=x[..., :8]), dict(k=x.half()), dict(k=x.double(), v=x.double()), dict(k=x[0]),
                                dict(keys=k8, values=k8.clone(), scales=(s, s)),
                                dict(keys=k8, values=k8.clone(), scales=tuple(t[:1].expand(6, 4, 3) for t in _scales()))])


def test_read_refuses(ge):
    k, v = _caches()
    ok = dict(keys=k, values=v, table=torch.zeros(2, 5, dtype=torch.int32), begin=[0, 3, 7])
    out = torch.zeros(7, 3, 16, dtype=BF)
    _refusals(ge.kv.read, ok, [*_bad_caches(), dict(table=ok["table"].long()), dict(table=ok["table"][0]), dict(table=ok["table"][:, :0]),
                               dict(table=torch.zeros(5, 2, dtype=torch.int32).t()), dict(begin=[0, 3]), dict(first=[0]), dict(dtype=I8),
                               dict(max_tokens=-1), dict(max_tokens=1 << 26), dict(out=(out, out)), dict(out=(out, out[:6])),
                               dict(out=(out, out.float())), dict(out=(out, torch.zeros(7, 16, 3, dtype=BF).transpose(1, 2)))])


def test_attend_refuses(ge):
    k, v = _caches()
    q = torch.zeros(7, 6, 16, dtype=BF)
    ok = dict(q=q, keys=k, values=v, table=torch.zeros(2, 5, dtype=torch.int32), seq_len=[9, 9], begin=[0, 3, 7])
    _refusals(ge.kv.attend, ok, [*_bad_caches(), dict(q=q.half()), dict(q=q.float()), dict(q=q[:, :4]), dict(q=q[:, :0]), dict(q=q[0]),
                                 dict(q=q[..., :8]), dict(table=ok["table"].float()), dict(seq_len=[9]), dict(begin=[0, 7]),
                                 dict(begin=None), dict(status=[0]), dict(begin=None, q=q[:2], max_new=2),
                                 dict(begin=None, q=q[:2], parents=[-1, -1]), dict(max_new=0), dict(max_new=1 << 25),
                                 dict(parents=[-1] * 6), dict(parents=[-1] * 7, max_new=65), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(out=q[:6]), dict(out=q.float()),
                                 dict(out=torch.zeros(6, 7, 16, dtype=BF).transpose(0, 1))])


def test_reorder_refuses(ge):
    c = torch.zeros(2, 6, 4, 3, 8)
    ok = dict(caches=c, table=torch.zeros(4, 5, dtype=torch.int32), seq_len=[3] * 4, parents=torch.zeros(2, 2, dtype=torch.int32))
    _refusals(ge.kv.reorder, ok, [dict(caches=c[0, 0]), dict(caches=c[:1].expand(2, 6, 4, 3, 8)), dict(caches=c[..., ::2]),
                                  dict(table=ok["table"][:3]), dict(table=ok["table"].long()), dict(seq_len=[3] * 3),
                                  dict(parents=torch.zeros(4)), dict(parents=torch.zeros((1, 33), dtype=torch.int32)),
                                  dict(first=[0]), dict(parents=[[0, 0]]), dict(caches=torch.zeros(1, 1, 1, 1).expand(1 << 24, 1, 1, 4))])


def test_select_refuses(ge):
    x, s = torch.zeros(6, 50), torch.zeros(2, 3)
    _refusals(ge.beam.select, dict(logits=x, scores=s, n=4),
              [dict(logits=x[:5]), dict(logits=x.double()), dict(logits=x[0]), dict(logits=x[:, :0]), dict(scores=s[0]), dict(scores=s.int()),
               dict(n=0), dict(n=65), dict(logits=torch.zeros(66, 5), scores=torch.zeros(2, 33)), dict(scores=s.tolist())])


def test_packed_structs_are_the_headers(ge):
    """The structs that kv and beam pack have the fields, sizes and places of the ctypes ones (which the header pins)."""
    lib, kinds = ge._lib, {4: {C.c_uint32: "I", C.c_float: "f"}, 8: {C.c_int64: "q", C.c_void_p: "Q"}}
    for packed, cls in ((ge.kv._CACHE, lib.KvCache), (ge.kv._WRITE, lib.KvRows), (ge.kv._READ, lib.KvRead), (ge.kv._ATTEND, lib.Attention),
                        (ge.kv._REORDER, lib.Reorder), (ge.beam._BEAMS, lib.Beams)):
        flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([IfqQ])", packed.format))
        assert packed.size == C.sizeof(cls) and len(flat) == len(cls._fields_)
        assert [kinds[C.sizeof(t)][t] for _, t in cls._fields_] == list(flat)
        raw = cls.from_buffer_copy(packed.pack(*range(1, len(flat) + 1)))
        assert [getattr(raw, f) for f, _ in cls._fields_] == list(range(1, len(flat) + 1))


def test_attend_refuses_more_rows_than_are_counted(ge):
    """New tokens times a head's query heads past 2^32."""
    k = torch.zeros((1, 1, 1, 8), dtype=BF)
    ok = dict(q=torch.zeros((1, 1, 8), dtype=BF).expand(1 << 24, 255, 8), keys=k, values=k.clone(), begin=[0, 1], max_new=1 << 24, seq_len=[1],
              table=torch.zeros((1, 1), dtype=torch.int32))
    _refusals(ge.kv.attend, ok, [dict(q=torch.zeros((1, 1, 8), dtype=BF).expand(1 << 24, hq, 8)) for hq in (256, 300, 512)])


def test_attend_refuses_scales_past_2_to_127(ge):
    """A scale times log2 e is to be finite in fp32."""
    k, v = _caches()
    ok = dict(q=torch.zeros(7, 6, 16, dtype=BF), keys=k, values=v, table=torch.zeros(2, 5, dtype=torch.int32), seq_len=[9, 9], begin=[0, 3, 7],
              scale=2.0 ** 127)
    _refusals(ge.kv.attend, ok, [dict(scale=s) for s in (3e38, -3e38, 2.0 ** 127 * 1.001, -1e300)])
