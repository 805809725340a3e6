"""What a step of forward.py refuses before anything reaches the device (its buffers are host memory here: nothing runs)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch


@pytest.fixture
def model(pkg):
    from pyodide_llm_amd import forward
    shape = SimpleNamespace(dim=64, hidden_dim=128, layers=1, heads=2, kv_heads=1, head_size=32)
    norms = {name: np.ones((1, 64), np.float32) for name in ("rms_att_weight", "rms_ffn_weight", "rms_final_weight")}
    ck = SimpleNamespace(torch=torch, shape=shape, device="cpu", dtype="int8", relaxed=True, vectors=norms, matrices={})
    return forward.Forward(ck, tokens=4, sequences=2, pages=4, width=2, page=16)


def step(model, **wrong):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    given = dict(x=torch.zeros(2, 64), starts=ints(0, 1, 2), lengths=ints(1, 1), table=torch.zeros(2, 2, dtype=torch.int32))
    given.update(wrong)
    return model.step(*given.values())


@pytest.mark.parametrize("wrong", [
    dict(x=torch.zeros(2, 64, dtype=torch.float16)), dict(x=torch.zeros(2, 64, dtype=torch.bfloat16)),
    dict(x=torch.zeros(2, 64, dtype=torch.float64)), dict(x=torch.zeros(2, 64, dtype=torch.int32)),
    dict(x=torch.zeros(2, 128)[:, ::2]), dict(x=torch.zeros(5, 64)), dict(x=torch.zeros(2, 32)), dict(x=torch.zeros(0, 64)),
    dict(x=torch.zeros(128)),
    # all of a step's tensors on another device than its buffers
    dict(x=torch.zeros(2, 64, device="meta"), starts=torch.zeros(3, dtype=torch.int32, device="meta"),
         lengths=torch.zeros(2, dtype=torch.int32, device="meta"), table=torch.zeros(2, 2, dtype=torch.int32, device="meta")),
    dict(starts=torch.zeros(3, dtype=torch.int32, device="meta")), dict(lengths=torch.ones(2, dtype=torch.int64)),
    dict(table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), dict(starts=torch.zeros(4, dtype=torch.int32)),
    dict(starts=torch.zeros(3, 2, dtype=torch.int32)), dict(lengths=torch.ones(2, 2, dtype=torch.int32)),
])
def test_step_refuses(model, wrong):
    with pytest.raises(ValueError, match="refused"):
        step(model, **wrong)
