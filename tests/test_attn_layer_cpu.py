"""AttnLayer / C3Attn without a GPU: state_dict surface, launch lists, pruned backwards, refused head layouts."""
import os

import pytest
import torch

from multiyolov5_amd import runtime as R
from multiyolov5_amd.models.common import C3, AttnLayer, C3Attn
from multiyolov5_amd.models.yolo import Model
from tests.util import CFG


def test_heads_are_checked():
    for c, h, kv in ((60, 4, 4), (64, 3, None), (64, 4, 3), (1024, 4, None), (20, 1, None)):
        with pytest.raises(ValueError):
            AttnLayer(c, h, kv)
    assert set(AttnLayer(64, 4).state_dict()) == {f'{n}.{p}' for n in ('norm1', 'norm2', 'qkv', 'proj', 'fc2') for p in ('weight', 'bias')} | {'fc1.weight'}
    assert isinstance(C3Attn(32, 64, 2, 2), C3) and len(C3Attn(32, 64, 2, 2).m) == 2


@pytest.mark.parametrize('dt', [torch.float16, torch.float32], ids=['fp16', 'fp32'])
def test_configuration_plans(dt):
    m = Model(os.path.join(CFG, 'yolov5s_city_seg_attn.yaml'))
    assert sum(isinstance(x, C3Attn) for x in m.modules()) == 2 and m.stride.tolist() == [8., 16., 32.]
    h = R.PlanHolder(m.train(), [torch.zeros(2, 3, 64, 128)], ('t', 0), dt, True)
    fwd = [c.name for o in h.plan.ops for c in o.fwd_calls]
    bwd = [c.name for o in h.plan.ops for c in o.bwd_calls]
    assert [fwd.count('myolo_' + n) for n in ('layernorm_fwd', 'rope', 'attn_fwd')] == [4, 2, 2]
    assert [bwd.count('myolo_' + n) for n in ('layernorm_bwd', 'rope', 'attn_bwd')] == [4, 2, 2]
    for live in ([0], [1], [3], [0, 1, 2]):
        sched = h.plan.bwd_schedule(live)
        assert isinstance(sched, list) and not h.plan.check_bwd_schedule(sched)
    h = R.PlanHolder(m.eval(), [torch.zeros(2, 3, 64, 128)], ('t', 0), dt, False)
    assert sum(c.name == 'myolo_attn_fwd' for o in h.plan.ops for c in o.fwd_calls) == 2 and not any(o.bwd_calls for o in h.plan.ops)
