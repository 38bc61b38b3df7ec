"""Dense and gated Dense over MXFP4 weights.

The reference has neither: its float Dense (``src/aie4ml/op_impls/families/matmul/resolver.py:110-127``) keeps lhs, rhs and
output in one float format.  Here ``mx_dense`` (what
``GraphBuilder.dense`` emits for weights of the ``MXFP4`` precision, ``qtypes.MXFP4``) reads a bfloat16 or
float32 activation, which the plan quantises to MXFP4 where it is read, multiplies on the tensor cores with float32
accumulation, and writes bfloat16 or float32.  ``gated_dense`` is the first half of a gated feed-forward block:
``act(x Wg + bg) * (x Wu + bu)``.  Between two such products the plan keeps the activation in MXFP4.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any, Dict

import numpy as np

from ..ir import ExecutionEntry, OpNode, input_tensor_for_role, optional_tensor_for_role
from ..qtypes import AIEDataType, FloatFormat, FloatIntent
from ..quant_utils import from_mx, to_mx
from .base import CUDA_GENERATIONS, FamilyResolver, OpImplVariant, family_resolver, register_variant
from .matmul import _transposed
from .precision import ACTIVATION_CODE, resolve_exact_storage_dtype
from .views import view_data, view_shape

_ACTIVATION_FORMATS = ('bfloat16', 'float32')


def _is_mx(tensor) -> bool:
    return isinstance(tensor.precision, FloatIntent) and tensor.precision.format is FloatFormat.MXFP4


def _precision(node: OpNode, weight_roles) -> Dict[str, AIEDataType]:
    out = {'output': resolve_exact_storage_dtype(node.outputs[0].precision, namespace='output', layer_name=node.name),
           'lhs': resolve_exact_storage_dtype(input_tensor_for_role(node, 'lhs').precision, namespace='lhs', layer_name=node.name)}
    for role in ('lhs', 'output'):
        if out[role].format not in _ACTIVATION_FORMATS:
            raise ValueError(f'{node.name}: {node.op_type} over MXFP4 weights needs a bfloat16 or float32 {role}, got '
                             f'{out[role].format!r}.')
    for role in weight_roles:
        if not _is_mx(input_tensor_for_role(node, role)):
            raise ValueError(f'{node.name}: {node.op_type} needs MXFP4 weights (role {role!r}).')
        out[role] = AIEDataType(format='mxfp4', frac=0)
    out['acc'] = AIEDataType(format='float32', frac=0)
    return out


def _pack_weights(node: OpNode, role: str):
    """-> (codes [N, pitch / 2], scale tiles, the float32 values [K, N] they stand for)"""
    W = view_data(node, input_tensor_for_role(node, role))
    K, N = int(W.shape[0]), int(W.shape[1])
    codes, tiles = to_mx(np.ascontiguousarray(W.T))
    return codes, tiles, np.ascontiguousarray(from_mx(codes, tiles, N, K).T)


def _pack_bias(node: OpNode, role: str):
    bias = optional_tensor_for_role(node, role)
    return None if bias is None else np.ascontiguousarray(np.asarray(bias.data, dtype=np.float32).reshape(-1))


@dataclass(frozen=True)
class MxDenseConfig:
    precision: Dict[str, AIEDataType]
    activation: str
    transpose_lhs: bool
    n_in: int
    n_out: int
    shift: int = 0
    accumulator_tag: str = 'accfloat'
    rounding_mode: str = 'conv_even'


def _refuse_views(node: OpNode, config: MxDenseConfig) -> None:
    if config.transpose_lhs:
        raise NotImplementedError(f'{node.name}: {node.op_type} over MXFP4 weights has no kernel for a transposed input view.')


def _check_bias(node: OpNode, role: str, n_out: int) -> None:
    bias = optional_tensor_for_role(node, role)
    if bias is not None and int(np.asarray(bias.data).size) != n_out:
        raise ValueError(f'{node.name}: {role} requires exactly {n_out} elements, got {int(np.asarray(bias.data).size)}.')


def _check_extents(node: OpNode, weight_shape, lhs_shape) -> None:
    """What the kernels are told (n_in, n_out, the output's rows and columns) is what the tensors hold."""
    given = tuple(node.metadata.get(key) for key in ('n_in', 'n_out'))
    if given != weight_shape:
        raise ValueError(f'{node.name}: n_in and n_out {given} do not match the weight {weight_shape}.')
    out = tuple(int(d) for d in node.outputs[0].shape)
    rows = math.prod(lhs_shape[:-1])
    if not out or out[-1] != weight_shape[1] or math.prod(out[:-1]) != rows:
        raise ValueError(f'{node.name}: output {out} does not hold {rows} x {weight_shape[1]} results of the input {lhs_shape}.')


def _check_activation(node: OpNode, known) -> None:
    if node.metadata.get('activation') not in known:
        raise ValueError(f"{node.name}: unknown activation {node.metadata.get('activation')!r}; one of {sorted(known)}.")


@family_resolver('mx_dense')
class MxDenseFamilyResolver(FamilyResolver):
    op_type = 'mx_dense'

    def validate_structure(self, node, _device) -> None:
        lhs_shape = tuple(view_shape(node, input_tensor_for_role(node, 'lhs'), 'inputs'))
        weight = input_tensor_for_role(node, 'rhs')
        shape = tuple(view_shape(node, weight, 'inputs'))
        if len(lhs_shape) < 2:
            raise ValueError(f'{node.name}: mx_dense requires a rank>=2 input, got {lhs_shape}.')
        if not weight.is_parameter or len(shape) != 2 or shape[0] != lhs_shape[-1]:
            raise ValueError(f'{node.name}: mx_dense needs a constant [K, N] weight that fits the input {lhs_shape}, got {shape}.')
        _check_extents(node, shape, lhs_shape)
        _check_bias(node, 'bias', shape[1])
        _check_activation(node, ('none', 'relu'))


@register_variant
class CudaMxDenseVariant(OpImplVariant):
    variant_id = 'mx_dense.cuda.v1'
    op_type = 'mx_dense'

    def matches(self, node: OpNode, device) -> bool:
        return device.generation in CUDA_GENERATIONS

    def resolve(self, node: OpNode, device, directives=None) -> MxDenseConfig:
        return MxDenseConfig(precision=_precision(node, ('rhs',)), activation=node.metadata['activation'],
                             transpose_lhs=_transposed(node, input_tensor_for_role(node, 'lhs')),
                             n_in=int(node.metadata['n_in']), n_out=int(node.metadata['n_out']))

    def validate_config(self, node: OpNode, config: MxDenseConfig, _device) -> None:
        _refuse_views(node, config)

    def pack(self, inst: ExecutionEntry) -> Dict[str, Any]:
        codes, tiles, values = _pack_weights(inst.node, 'rhs')
        return {'weights_kn': values, 'packed_weights': codes, 'packed_scales': tiles, 'packed_bias': _pack_bias(inst.node, 'bias')}

    def plan_op(self, inst: ExecutionEntry) -> Dict[str, Any]:
        node, cfg = inst.node, inst.config
        has_bias = optional_tensor_for_role(node, 'bias') is not None
        return {'kind': 'dense_mx', 'name': node.name, 'lhs': input_tensor_for_role(node, 'lhs').name, 'out': node.outputs[0].name,
                'weight': f'{node.name}/weights', 'bias': f'{node.name}/bias' if has_bias else None, 'K': cfg.n_in, 'N': cfg.n_out,
                'relu': cfg.activation == 'relu', 'dtype': cfg.precision['output'].format}


@family_resolver('gated_dense')
class GatedDenseFamilyResolver(FamilyResolver):
    op_type = 'gated_dense'

    def validate_structure(self, node, _device) -> None:
        lhs_shape = tuple(view_shape(node, input_tensor_for_role(node, 'lhs'), 'inputs'))
        gate, up = input_tensor_for_role(node, 'gate'), input_tensor_for_role(node, 'up')
        if len(lhs_shape) < 2:
            raise ValueError(f'{node.name}: gated_dense requires a rank>=2 input, got {lhs_shape}.')
        if not gate.is_parameter or not up.is_parameter:
            raise NotImplementedError(f'{node.name}: gated_dense needs constant weights.')
        shape, up_shape = (tuple(view_shape(node, t, 'inputs')) for t in (gate, up))
        if len(shape) != 2 or shape != up_shape or shape[0] != lhs_shape[-1]:
            raise ValueError(f'{node.name}: gated_dense weights {shape} and {up_shape} do not fit the input {lhs_shape}.')
        _check_extents(node, shape, lhs_shape)
        for role in ('gate_bias', 'up_bias'):
            _check_bias(node, role, shape[1])
        _check_activation(node, ACTIVATION_CODE)


@register_variant
class CudaMxGatedDenseVariant(OpImplVariant):
    variant_id = 'gated_dense.mx.cuda.v1'
    op_type = 'gated_dense'

    def matches(self, node: OpNode, device) -> bool:
        return device.generation in CUDA_GENERATIONS

    def resolve(self, node: OpNode, device, directives=None) -> MxDenseConfig:
        return MxDenseConfig(precision=_precision(node, ('gate', 'up')), activation=node.metadata['activation'],
                             transpose_lhs=_transposed(node, input_tensor_for_role(node, 'lhs')),
                             n_in=int(node.metadata['n_in']), n_out=int(node.metadata['n_out']))

    def validate_config(self, node: OpNode, config: MxDenseConfig, _device) -> None:
        _refuse_views(node, config)

    def pack(self, inst: ExecutionEntry) -> Dict[str, Any]:
        out = {}
        for role in ('gate', 'up'):
            codes, tiles, values = _pack_weights(inst.node, role)
            out.update({f'{role}_kn': values, f'packed_{role}': codes, f'packed_{role}_scales': tiles,
                        f'packed_{role}_bias': _pack_bias(inst.node, f'{role}_bias')})
        return out

    def plan_op(self, inst: ExecutionEntry) -> Dict[str, Any]:
        node, cfg = inst.node, inst.config
        op = {'kind': 'gated_dense_mx', 'name': node.name, 'lhs': input_tensor_for_role(node, 'lhs').name, 'out': node.outputs[0].name,
              'K': cfg.n_in, 'N': cfg.n_out, 'activation': cfg.activation, 'dtype': cfg.precision['output'].format}
        for role in ('gate', 'up'):
            op[role] = f'{node.name}/{role}'
            op[f'{role}_bias'] = f'{node.name}/{role}_bias' if optional_tensor_for_role(node, f'{role}_bias') is not None else None
        return op
