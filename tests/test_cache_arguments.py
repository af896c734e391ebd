"""Numbers that the C interface holds in 32 bits are refused by the Python calls when they do not fit, instead of being
taken modulo 2^32 (sinks = -1 would be every key, a layer 2^32 layer 0). No GPU needed."""
import pytest

import backburner_b200 as pa
from backburner_b200 import api


class _Cache:
    n_layers, nkv, hd, device = 3, 8, 128, 0


@pytest.mark.parametrize("name", ["n_sets", "n_tok", "gqa", "max_pages", "window", "sinks"])
@pytest.mark.parametrize("value", [-1, -(1 << 32), 1 << 32, (1 << 32) + 1])
def test_plan_sizes(name, value):
    kw = dict(n_sets=1, n_tok=1, gqa=5, max_pages=4, window=64, sinks=4)
    kw[name] = value
    with pytest.raises(pa.PaCudaError) as e:
        pa.CachePlan(None, _Cache, **kw)
    assert e.value.code == api.EINVAL and f"{name} = {value}" in str(e.value)


def test_plan_rows():
    with pytest.raises(pa.PaCudaError) as e:
        pa.CachePlan(None, _Cache, n_sets=1, n_tok=1 << 20, gqa=1 << 20, max_pages=4)
    assert e.value.code == api.EINVAL and "rows" in str(e.value)


@pytest.mark.parametrize("layer", [-1, 3, 1 << 32, -(1 << 32)])
def test_layers(layer):
    with pytest.raises(pa.PaCudaError) as e:
        api._layer(_Cache, layer)
    assert e.value.code == api.EINVAL and str(layer) in str(e.value)
    assert [api._layer(_Cache, i) for i in range(3)] == [0, 1, 2]
