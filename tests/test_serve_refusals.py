"""What an Adapters of factors refuses before anything is computed, and what a Serving needs of its Forward."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch


def pair(a=(2, 3, 8, 64), b=(2, 3, 96, 8), kind=torch.float16):
    return torch.zeros(a, dtype=kind), torch.zeros(b, dtype=kind)


@pytest.mark.parametrize("factors, scales", [
    ({}, None), ({"wq": pair(kind=torch.float32)}, None), ({"wq": pair(a=(2, 3, 12, 64), b=(2, 3, 96, 12))}, None),
    ({"wq": pair(a=(3, 8, 64))}, None), ({"wq": pair(b=(2, 3, 96, 16))}, None), ({"wq": pair(b=(1, 3, 96, 8))}, None),
    ({"wq": pair(b=(2, 2, 96, 8))}, None), ({"wq": pair(a=(2, 3, 8, 72))}, None),
    ({"wq": pair(), "wk": pair(kind=torch.bfloat16)}, None), ({"wq": (pair()[0], pair()[1].transpose(0, 1).contiguous().transpose(0, 1))}, None),
    ({"wq": pair()}, torch.ones(2)), ({"wq": pair()}, torch.ones(3, dtype=torch.float64)), ({"wq": pair()}, torch.ones(6)[::2]),
    ({"wq": pair(a=(2, 3, 264, 64), b=(2, 3, 96, 264))}, None)])
def test_adapters_refuse(pkg, factors, scales):
    from pyodide_llm_amd import adapters
    with pytest.raises(ValueError, match="refused"):
        adapters.Adapters(factors, scales)


def test_adapters_hold(pkg):
    from pyodide_llm_amd import adapters
    held = adapters.Adapters({"wq": pair()}, torch.ones(3))
    y = torch.zeros(5, 96)
    target = held.target("wq", 1, y, 384)
    a, b = held.factors["wq"]
    assert (held.count, held.rank, held.form, target.rows) == (3, 8, 1, 96)
    assert (target.a, target.b, target.y) == (a[1].data_ptr(), b[1].data_ptr(), y.data_ptr())


def test_serving_refuses_more_places_than_rows(pkg):
    from pyodide_llm_amd import serve
    with pytest.raises(ValueError, match="refused"):
        serve.Serving(SimpleNamespace(torch=torch, sequences=5, tokens=4, y=torch.zeros(4, 64)))


@pytest.mark.parametrize("name, a, b", [("wq", (1, 3, 8, 32), (1, 3, 64, 8)), ("wq", (2, 3, 8, 64), (2, 3, 64, 8)),
                                        ("wq", (1, 3, 8, 64), (1, 3, 96, 8)), ("token_embedding_table", (1, 3, 8, 64), (1, 3, 64, 8)),
                                        ("w9", (1, 3, 8, 64), (1, 3, 64, 8))])
def test_serving_refuses_adapters_of_another_model(pkg, name, a, b):
    """when it is made, not by a step that has moved lengths and pages on"""
    from pyodide_llm_amd import adapters, forward, serve
    shape = SimpleNamespace(dim=64, hidden_dim=128, layers=1, heads=2, kv_heads=2, head_size=32, vocab=100)
    norms = {n: np.ones((1, 64), np.float32) for n in ("rms_att_weight", "rms_ffn_weight", "rms_final_weight")}
    matrices = {n: SimpleNamespace(layers=1, n=64, rows=64) for n in ("wq", "wk", "token_embedding_table")}
    ck = SimpleNamespace(torch=torch, shape=shape, device="cpu", dtype="int8", relaxed=True, vectors=norms, matrices=matrices)
    model = forward.Forward(ck, tokens=4, sequences=2, pages=4, width=2, page=16)
    serve.Serving(model, adapters.Adapters({"wq": pair((1, 3, 8, 64), (1, 3, 64, 8))}))
    with pytest.raises(ValueError, match="refused"):
        serve.Serving(model, adapters.Adapters({name: pair(a, b)}))
