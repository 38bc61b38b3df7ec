"""Graphs whose MXFP4 nodes contradict their tensors are refused before any launch exists (CPU)."""

import contextlib

import numpy as np
import pytest

from aie4ml_b200 import from_graph
from aie4ml_b200.runtime import Plan

F32 = {'float': 'float32'}
MX = {'float': 'mxfp4'}


def dense_spec(**change):
    """x [6, 64] -> 40 features; the metadata and the output's shape as given."""
    rng = np.random.default_rng(0)
    meta = {'n_in': 64, 'n_out': 40, 'activation': 'none'}
    meta.update({k: v for k, v in change.items() if k != 'shape'})
    return {'name': 'g', 'inputs': [{'name': 'x', 'shape': [6, 64], 'precision': F32}],
            'params': {'w': {'data': rng.normal(size=(64, 40)), 'precision': MX}},
            'nodes': [{'name': 'fc', 'op': 'mx_dense', 'inputs': ['x', 'w'], 'roles': ['lhs', 'rhs'], 'metadata': meta,
                       'outputs': [{'name': 'y', 'shape': change.get('shape', [6, 40]), 'precision': F32}]}], 'outputs': ['y']}


def block_spec(hidden=(300, 96), **change):
    """x [300, 64] -> gated 96 -> 64; `hidden` is the shape stated for the tensor between the two products."""
    rng = np.random.default_rng(0)
    meta = {'n_in': 64, 'n_out': 96, 'activation': 'silu'}
    meta.update(change)
    return {'name': 'g', 'inputs': [{'name': 'x', 'shape': [300, 64], 'precision': F32}],
            'params': {n: {'data': rng.normal(size=s), 'precision': MX} for n, s in (('wg', (64, 96)), ('wu', (64, 96)), ('wd', (96, 64)))},
            'nodes': [{'name': 'gu', 'op': 'gated_dense', 'inputs': ['x', 'wg', 'wu'], 'roles': ['lhs', 'gate', 'up'], 'metadata': meta,
                       'outputs': [{'name': 'h', 'shape': list(hidden), 'precision': F32}]},
                      {'name': 'down', 'op': 'mx_dense', 'inputs': ['h', 'wd'], 'roles': ['lhs', 'rhs'],
                       'metadata': {'n_in': 96, 'n_out': 64, 'activation': 'none'},
                       'outputs': [{'name': 'y', 'shape': [hidden[0], 64], 'precision': F32}]}], 'outputs': ['y']}


def test_consistent_graphs_lower():
    assert [op['kind'] for op in from_graph(dense_spec()).export_plan()['ops']] == ['dense_mx']
    assert [op['kind'] for op in from_graph(dense_spec(shape=[2, 3, 40])).export_plan()['ops']] == ['dense_mx']   # rows may be split up
    assert [op['kind'] for op in from_graph(block_spec()).export_plan()['ops']] == ['gated_dense_mx', 'dense_mx']


@pytest.mark.parametrize('change', [{'n_in': 40}, {'n_in': 96}, {'n_out': 24}, {'n_out': 64}, {'n_in': None}])
def test_metadata_that_contradicts_the_weight(change):
    with pytest.raises(ValueError, match='fc: n_in and n_out .* do not match the weight'):
        from_graph(dense_spec(**change)).export_plan()
    with pytest.raises(ValueError, match='gu: n_in and n_out .* do not match the weight'):
        from_graph(block_spec(**change)).export_plan()


@pytest.mark.parametrize('shape', [[6, 41], [6, 32], [5, 40], [40], [1, 40], [12, 20]])
def test_output_that_does_not_hold_the_results(shape):
    with pytest.raises(ValueError, match='fc: output .* does not hold 6 x 40 results'):
        from_graph(dense_spec(shape=shape)).export_plan()


@pytest.mark.parametrize('hidden', [(1, 96), (128, 96), (301, 96), (300, 64), (300, 128)])
def test_hidden_tensor_that_does_not_hold_the_results(hidden):
    with pytest.raises(ValueError, match='gu: output .* does not hold 300 x 96 results'):
        from_graph(block_spec(hidden)).export_plan()


@pytest.fixture
def plan_on_cpu(monkeypatch):
    """Builds a plan's launch list in host memory; nothing is launched."""
    import torch

    monkeypatch.setattr(torch.cuda, 'is_available', lambda: True)
    monkeypatch.setattr(torch.cuda, 'device', lambda _device: contextlib.nullcontext())
    return lambda model: Plan(model.run_pipeline().context, device='cpu')


def test_plan_holds_each_launch_to_its_buffers(plan_on_cpu):
    plan = plan_on_cpu(from_graph(block_spec()))
    assert [op['kind'] for op in plan.ops] == ['quantize_mx', 'gated_dense_mx', 'dense_mx']
    assert [args[-4:-1] for _, args in plan.launches[1:]] == [(300, 64, 96), (300, 96, 64)]      # rows, K, features


@pytest.mark.parametrize('tensor,shape,match', [('h', (1, 96), 'gu: results of .300, 96. do not fit'), ('h', (300, 64), 'gu: results of .300, 96. do not fit'),
                                                ('x', (300, 32), 'gu: input of 32 features for weights of 64'), ('y', (300, 32), 'down: shape mismatch')])
def test_plan_refuses_what_does_not_fit(plan_on_cpu, tensor, shape, match):
    """The plan's own comparison, for a graph that changed after it was lowered."""
    model = from_graph(block_spec()).run_pipeline()
    model.context.ir.logical.tensors[tensor].shape = shape
    with pytest.raises(ValueError, match=match):
        plan_on_cpu(model)


def test_plan_refuses_packed_weights_of_another_size(plan_on_cpu):
    model = from_graph(block_spec()).run_pipeline()
    entry = model.context.ir.execution.get('down')
    entry.artifacts['packed_weights'] = entry.artifacts['packed_weights'][:-1]
    with pytest.raises(ValueError, match='down: packed weights .* are not 64 rows of 96 values'):
        plan_on_cpu(model)
