"""A Transpose of a constant weight: the packed weights are those the node sees (CPU)."""

import numpy as np
import pytest

from aie4ml_b200 import from_graph

F32, BF16, MX, INT8 = {'float': 'float32'}, {'float': 'bfloat16'}, {'float': 'mxfp4'}, {'width': 8, 'frac': 4}


def lowered(op, precision, weight_precision, k, n, transposed):
    rng = np.random.default_rng(0)
    w, w2 = (rng.normal(size=(k, n)) for _ in range(2))
    roles = ['lhs', 'gate', 'up'] if op == 'gated_dense' else ['lhs', 'rhs']
    params = {'w': {'data': w.T if transposed else w, 'precision': weight_precision}}
    nodes = []
    if transposed:
        nodes.append({'name': 't', 'op': 'transpose', 'inputs': ['w'], 'outputs': [{'name': 'wt', 'shape': [k, n], 'precision': weight_precision}],
                      'metadata': {'perm': [1, 0]}})
    ins = ['x', 'wt' if transposed else 'w']
    if op == 'gated_dense':
        params['w2'] = {'data': w2, 'precision': weight_precision}
        ins.append('w2')
    nodes.append({'name': 'fc', 'op': op, 'inputs': ins, 'roles': roles, 'metadata': {'n_in': k, 'n_out': n, 'activation': 'none'},
                  'outputs': [{'name': 'y', 'shape': [4, n], 'precision': precision}]})
    spec = {'name': 'g', 'inputs': [{'name': 'x', 'shape': [4, k], 'precision': precision}], 'params': params, 'nodes': nodes, 'outputs': ['y']}
    model = from_graph(spec).run_pipeline()
    return model.export_plan(), model.context.ir.execution.get('fc').artifacts


@pytest.mark.parametrize('op,precision,weight_precision', [('dense', INT8, INT8), ('dense', F32, F32), ('dense', BF16, BF16), ('mx_dense', F32, MX),
                                                           ('gated_dense', BF16, MX)])
@pytest.mark.parametrize('k,n', [(32, 32), (64, 48)])
def test_transposed_constant(op, precision, weight_precision, k, n):
    plain, packed = lowered(op, precision, weight_precision, k, n, False)
    seen, seen_packed = lowered(op, precision, weight_precision, k, n, True)
    assert plain['params'].keys() == seen['params'].keys()
    assert all(np.array_equal(plain['params'][key], seen['params'][key]) for key in plain['params'])
    assert packed.keys() == seen_packed.keys()
    assert all(np.array_equal(packed[key], seen_packed[key]) for key in packed if packed[key] is not None)
