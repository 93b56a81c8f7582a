"""Token operators: sizes that the kernels' 32-bit counters or one launch cannot hold are refused on the host (no GPU: nothing here reaches a launch)."""
import ctypes as C

import pytest
import torch

from multiyolov5_amd import _lib as L
from multiyolov5_amd.utils import tokens as T
from tests.test_tokens_cpu import EINVAL, FAKE, attn_desc, lib, rope_desc, rows  # noqa: F401 (lib: a fixture)


def test_layer_norm_channels(lib):  # noqa: F811
    c = (1 << 29) + 1
    x = rows(w=1, c=c)
    assert lib.myolo_layernorm_fwd(C.byref(x), None, None, 1e-5, C.byref(x), None, None) == EINVAL
    assert lib.myolo_layernorm_bwd(C.byref(x), C.byref(x), FAKE, None, None, 0, FAKE, FAKE, 0, FAKE, 1 << 50, None) == EINVAL
    with pytest.raises(L.MyoloError, match='channels'):
        T._ext().layer_norm(torch.zeros(1).expand(c), None, None, 1e-5)


def test_rotary_token(lib):  # noqa: F811
    for kw in (dict(hq=1 << 27), dict(hq=(1 << 31) - 1, hk=(1 << 31) - 1), dict(hk=1 << 30)):
        assert lib.myolo_rope(C.byref(rope_desc(**kw)), None) == EINVAL, kw
    with pytest.raises(L.MyoloError, match='rotary pairs'):
        T.rope_table((1 << 40, 1))


def test_attention_launches(lib):  # noqa: F811
    # 2^22 (batch, head) pairs of 8 blocks of 128 queries: 2^25 workgroups of 256 threads
    for kw in (dict(lq=1024), dict(lq=1, lk=1024)):
        d = attn_desc(b=1 << 16, hq=64, hk=64, ws=FAKE, ws_bytes=1 << 60, **kw)
        assert 'lk' in kw or lib.myolo_attn_fwd(C.byref(d), None) == EINVAL
        assert lib.myolo_attn_bwd(C.byref(d), None) == EINVAL
