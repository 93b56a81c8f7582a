"""Token operators without a GPU: descriptor layouts, what the C entries refuse before any launch, the rotary table, refusal of CPU tensors."""
import ctypes as C
import math
import os
import shutil
import subprocess
import tempfile

import pytest
import torch

from multiyolov5_amd import _lib as L
from multiyolov5_amd.utils import tokens as T
from tests.util import ROOT

EINVAL = -22


@pytest.fixture(scope='module')
def lib():
    from multiyolov5_amd import build
    build.build(verbose=False)
    return L.lib()


@pytest.mark.skipif(not shutil.which('gcc'), reason='no C compiler')
def test_descriptor_layouts():
    fields = {'myolo_rope_desc': (L.RopeDesc, ['pos', 'axis', 'qs', 'ps', 'b', 'dtype']),
              'myolo_attn_desc': (L.AttnDesc, ['o_res', 'lse', 'go', 'ws', 'ws_bytes', 'qs', 'gvs', 'b', 'sinks', 'scale'])}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "myolo.h"\nint main(void){\n'
    want = []
    for name, (cls, fs) in fields.items():
        src += f'printf("%zu ", sizeof({name}));\n' + ''.join(f'printf("%zu ", offsetof({name}, {f}));\n' for f in fs)
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f in fs]
    src += 'printf("%d %d %d\\n", MYOLO_ROPE_MAX_PAIRS, MYOLO_ROPE_MAX_AXES, MYOLO_ATTN_MAX_LEN);return 0;}\n'
    want += [L.ROPE_MAX_PAIRS, L.ROPE_MAX_AXES, L.ATTN_MAX_LEN]
    with tempfile.TemporaryDirectory() as td:
        with open(os.path.join(td, 'a.c'), 'w') as f:
            f.write(src)
        subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), os.path.join(td, 'a.c'), '-o', os.path.join(td, 'a')])
        got = [int(v) for v in subprocess.check_output([os.path.join(td, 'a')]).split()]
    assert got == want


FAKE = 1 << 20          # a pointer that is never followed: every call below is refused on the host


def rows(n=1, h=1, w=4, c=16, dtype=L.F16, ptr=FAKE):
    return L.Tensor(ptr, n, h, w, c, h * w * c, w * c, c, dtype, 0)


def test_layernorm_refusals(lib):
    def fwd(x, o, eps=1e-5):
        return lib.myolo_layernorm_fwd(C.byref(x) if x else None, None, None, eps, C.byref(o) if o else None, None, None)
    assert fwd(rows(w=0), rows(w=0)) == 0                                           # no rows: nothing to do
    for a in ((None, rows()), (rows(), None), (rows(), rows(c=8)), (rows(), rows(dtype=L.F32)), (rows(c=0), rows(c=0)), (rows(ptr=0), rows()),
              (rows(dtype=L.U8), rows(dtype=L.U8)), (rows(n=-1), rows(n=-1)), (rows(), rows(w=5)), (rows(h=1 << 20, w=1 << 20), rows(h=1 << 20, w=1 << 20)),
              (rows(), rows(), -1.0), (rows(), rows(), math.nan)):
        assert fwd(*a) == EINVAL, a

    def bwd(go=rows(), x=rows(), saved=FAKE, gx=None, dg=0, ws=0, nb=0):
        return lib.myolo_layernorm_bwd(C.byref(go), C.byref(x), saved, None, C.byref(gx) if gx else None, 0, dg, None, 0, ws, nb, None)
    need = lib.myolo_layernorm_ws_bytes(4, 16)
    assert need > 0 and lib.myolo_layernorm_ws_bytes(0, 16) == 0 and lib.myolo_layernorm_ws_bytes(4, 0) == 0
    for kw in (dict(go=rows(w=3)), dict(saved=None, gx=rows()), dict(gx=rows(c=8)), dict(dg=FAKE), dict(dg=FAKE, ws=FAKE, nb=need - 1),
               dict(dg=FAKE, ws=FAKE + 4, nb=need)):
        assert bwd(**kw) == EINVAL, kw


def rope_desc(**kw):
    d = L.RopeDesc()
    d.q = d.qo = d.k = d.ko = d.pos = FAKE
    tab = T.rope_table((4, 4))
    d._keep = tab
    d.turns, d.axis = C.cast(tab[0], C.c_void_p), C.cast(tab[1], C.c_void_p)
    d.b, d.l, d.hq, d.hk, d.d, d.npair, d.naxis, d.dtype = 1, 3, 2, 1, 16, 8, 2, L.F16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_rope_refusals(lib):
    assert lib.myolo_rope(C.byref(rope_desc(l=0, q=0)), None) == 0
    for kw in (dict(q=0), dict(ko=0), dict(k=0), dict(pos=0), dict(turns=0), dict(axis=0), dict(d=15), dict(npair=-1), dict(naxis=1), dict(naxis=5),
               dict(naxis=0), dict(hq=0), dict(hk=-1), dict(b=-1), dict(dtype=L.U8), dict(npair=129, d=300)):
        assert lib.myolo_rope(C.byref(rope_desc(**kw)), None) == EINVAL, kw
    assert lib.myolo_rope(None, None) == EINVAL


def attn_desc(**kw):
    d = L.AttnDesc()
    d.q = d.k = d.v = d.o = d.go = d.gq = d.gk = d.gv = d.lse = FAKE
    d.b, d.lq, d.lk, d.hq, d.hk, d.d, d.dtype, d.scale = 1, 64, 64, 4, 2, 64, L.F16, 0.125
    for n in ('qs', 'os', 'gos', 'gqs'):
        setattr(d, n, (C.c_int64 * 3)(64 * 256, 256, 64))
    for n in ('ks', 'vs', 'gks', 'gvs'):
        setattr(d, n, (C.c_int64 * 3)(64 * 128, 128, 64))
    for k, v in kw.items():
        setattr(d, k, (C.c_int64 * 3)(*v) if isinstance(v, tuple) else v)
    return d


def test_attention_refusals(lib):
    shape = [dict(hk=3), dict(hq=0), dict(hk=0), dict(d=12), dict(d=0), dict(d=136), dict(dtype=L.U8), dict(window=-1), dict(sinks=-1), dict(lq=-1), dict(b=-1),
             dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(lk=(1 << 28) + 1), dict(window=(1 << 28) + 1), dict(lq=(1 << 28)), dict(b=1 << 23),
             dict(q=FAKE + 2), dict(q=0), dict(o=0), dict(k=0), dict(v=FAKE + 8), dict(ks=(64 * 128, 130, 64)), dict(os=(64 * 256, 256, 63)), dict(o_res=FAKE + 2)]
    for kw in shape:
        d = attn_desc(**kw)
        assert lib.myolo_attn_fwd(C.byref(d), None) == EINVAL, kw
        d.ws, d.ws_bytes = FAKE, 1 << 40
        assert lib.myolo_attn_bwd(C.byref(d), None) == EINVAL, kw
    assert lib.myolo_attn_fwd(None, None) == EINVAL and lib.myolo_attn_bwd(None, None) == EINVAL
    # one query over a long cache is split: without scratch, with too little, with scratch off a 16-byte boundary
    d = attn_desc(lq=1, lk=32768)
    need = lib.myolo_attn_ws_bytes(C.byref(d), 0)
    assert need > 0
    for ws, nb in ((0, 0), (FAKE, need - 1), (FAKE + 4, need)):
        d.ws, d.ws_bytes = ws, nb
        assert lib.myolo_attn_fwd(C.byref(d), None) == EINVAL
    for kw in (dict(), dict(ws=FAKE, ws_bytes=64 * 4 * 4 - 1), dict(ws=FAKE + 8, ws_bytes=1 << 20), dict(ws=FAKE, ws_bytes=1 << 20, gk=0),
               dict(ws=FAKE, ws_bytes=1 << 20, go=0), dict(ws=FAKE, ws_bytes=1 << 20, lse=0), dict(ws=FAKE, ws_bytes=1 << 20, gq=FAKE + 2)):
        assert lib.myolo_attn_bwd(C.byref(attn_desc(**kw)), None) == EINVAL, kw
    assert lib.myolo_attn_ws_bytes(C.byref(attn_desc(hk=3)), 0) == 0
    # nothing to do
    assert lib.myolo_attn_fwd(C.byref(attn_desc(b=0)), None) == 0 and lib.myolo_attn_fwd(C.byref(attn_desc(lq=0)), None) == 0
    assert lib.myolo_attn_bwd(C.byref(attn_desc(b=0)), None) == 0 and lib.myolo_attn_bwd(C.byref(attn_desc(gq=0, gk=0, gv=0)), None) == 0


def test_rope_table():
    turns, axis = T.rope_table((1, 2, 3), 10000.0, 'shared')
    assert list(axis) == [0, 1, 1, 2, 2, 2]
    assert all(abs(t * 2 * math.pi - 10000.0 ** -(j / 6)) <= 1e-15 for j, t in enumerate(turns))
    turns, axis = T.rope_table((0, 2, 2), 100.0, 'axis')
    assert list(axis) == [1, 1, 2, 2]
    assert all(abs(t * 2 * math.pi - f) <= 1e-15 for t, f in zip(turns, (1.0, 0.1, 1.0, 0.1)))


def test_autograd_nodes_load_and_raise_the_frameworks_error(lib):
    ext = T._ext()
    assert ext is T._ext()
    with pytest.raises(L.MyoloError, match='no channels'):
        ext.layer_norm(torch.zeros(3, 0), None, None, 1e-5)
    q = torch.zeros(1, 2, 3, 16)
    with pytest.raises(L.MyoloError, match='3 query heads over 2 key heads'):
        ext.window_attention(q, q[:, :, :2], q[:, :, :2], 0, 0, False, None, None, None)


def test_cpu_tensors_are_refused():
    q, pos = torch.zeros(1, 2, 2, 16), torch.zeros(2, 1, dtype=torch.int64)
    for f in (lambda: T.layer_norm(q), lambda: T.rope_axes(q, q, pos, (8,)), lambda: T.window_attention(q, q, q)):
        with pytest.raises(L.MyoloError, match='no CPU path'):
            f()
