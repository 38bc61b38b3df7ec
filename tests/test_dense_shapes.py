"""Dense nodes that would read past their weight or bias are refused when they are lowered (CPU)."""

import numpy as np
import pytest

from aie4ml_b200 import from_graph

INT8 = {'width': 8, 'frac': 4}


def spec(precision, bias_size=None, **meta):
    rng = np.random.default_rng(0)
    params = {'w': {'data': rng.normal(size=(64, 40)), 'precision': precision}}
    ins, roles = ['x', 'w'], ['lhs', 'rhs']
    if bias_size is not None:
        params['b'] = {'data': rng.normal(size=bias_size), 'precision': precision if 'width' in precision else None}
        ins, roles = ins + ['b'], roles + ['bias']
    return {'name': 'g', 'inputs': [{'name': 'x', 'shape': [6, 64], 'precision': precision}], 'params': params,
            'nodes': [{'name': 'fc', 'op': 'dense', 'inputs': ins, 'roles': roles,
                       'metadata': dict({'n_in': 64, 'n_out': 40, 'use_bias': bias_size is not None}, **meta),
                       'outputs': [{'name': 'y', 'shape': [6, meta.get('n_out', 40)], 'precision': precision}]}], 'outputs': ['y']}


@pytest.mark.parametrize('precision,kind', [(INT8, 'dense'), ({'width': 16, 'frac': 8}, 'dense'), ({'float': 'bfloat16'}, 'dense_f'), ({'float': 'float32'}, 'dense_f')])
def test_dense_extents(precision, kind):
    assert from_graph(spec(precision)).export_plan()['ops'][0]['kind'] == kind
    assert from_graph(spec(precision, 40)).export_plan()['ops'][0]['bias'] == 'fc/bias'
    assert from_graph(spec(precision, n_out=32)).export_plan()['ops'][0]['N'] == 32      # the first columns alone: inside the weight
    for n_out in (41, 64):
        with pytest.raises(ValueError, match=f'fc: n_out {n_out} exceeds the 40 columns of the weight'):
            from_graph(spec(precision, n_out=n_out)).export_plan()
    for size in (1, 39):
        with pytest.raises(ValueError, match=f'fc: bias has {size} elements for 40 outputs'):
            from_graph(spec(precision, size)).export_plan()
