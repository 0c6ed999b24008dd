"""Momentum rule that orthogonalises what it subtracts, for weight matrices
beside (or instead of) a Kronecker-factored block: a layer that the
``constructor`` of ``KFAC`` gives no block, for instance."""

import math

import torch

from chainerkfac_b200 import ops
from chainerkfac_b200.optimizers import _base


class OrthogonalUpdateRule(_base.UpdateRule):
    """v = momentum v + g, and W = (1 - lr decay) W - lr s O, where O is
    ``ops.orthogonalize`` of g + momentum v (``nesterov``) or v, and s is
    ``scale`` or by default sqrt(max(1, rows / columns)).  The gradient g is
    ``param.kfgrad`` where a block has left one, else ``param.grad``.

    Takes the place of a parameter's rule, whose learning rate and momentum it
    goes on with::

        for p in matrices:
            p.update_rule = OrthogonalUpdateRule(optimizer.hyperparam)

    ``KFAC.update`` orthogonalises the matrices of all such rules together.
    ``DistributedKFAC`` exchanges the gradients of blocks only, and refuses
    the rule for a parameter without one.  Float32 weights of two dimensions
    and more (filters are rows)."""

    def __init__(self, parent_hyperparam=None, nesterov=True, steps=5,
                 coefficients=ops.NEWTON_SCHULZ, eps=1e-7, decay=0.0,
                 scale=None):
        if parent_hyperparam is None:
            from chainerkfac_b200.optimizers.kfac import _default_hyperparam
            parent_hyperparam = _default_hyperparam
        super(OrthogonalUpdateRule, self).__init__(parent_hyperparam)
        self.nesterov = nesterov
        self.steps = steps
        self.coefficients = coefficients
        self.eps = eps
        self.decay = decay
        self.scale = scale

    @staticmethod
    def check(param):
        """Refuses a weight that the rule's kernels do not take."""
        w = param.data
        if w.dim() < 2:
            raise ValueError('%s has %d dimension(s): only matrices can be '
                             'orthogonalised' % (param.name, w.dim()))
        if w.dtype != torch.float32:
            raise TypeError('%s is %s: the rule takes float32 weights'
                            % (param.name, w.dtype))
        if not w.is_contiguous():
            raise ValueError('%s must be contiguous' % param.name)

    def init_state(self, param):
        self.state['v'] = torch.zeros_like(param.data)

    def _scale_of(self, w):
        if self.scale is not None:
            return float(self.scale)
        rows = w.shape[0]
        return math.sqrt(max(1.0, rows * rows / float(w.numel())))

    def _settings(self):
        """What rules that are applied together have in common."""
        h, c = self.hyperparam, self.coefficients
        if hasattr(c[0], '__len__'):
            c = tuple(tuple(r) for r in c)
        return (h.lr, h.momentum, self.nesterov, self.steps, tuple(c),
                self.eps, self.decay)

    def prepare(self, param):
        self.check(param)
        super(OrthogonalUpdateRule, self).prepare(param)
        if param._loss_scale is not None and \
                getattr(param, 'kfgrad', None) is not None:
            param.kfgrad /= param._loss_scale

    def update_core(self, param):
        apply_rules([(self, param)])


def _gradient(param):
    g = getattr(param, 'kfgrad', None)
    return param.grad if g is None else g


def apply_rules(pairs):
    """``update_core`` of (rule, parameter) pairs, those with the same settings
    in one call."""
    groups = {}
    for rule, param in pairs:
        g = _gradient(param)
        if g is not None:
            groups.setdefault(rule._settings(), []).append(
                (rule, param, g.contiguous()))
    for (lr, momentum, nesterov, steps, coef, eps, decay), group in \
            groups.items():
        gs = [g for _, _, g in group]
        vs = [rule.state['v'] for rule, _, _ in group]
        us = vs
        ops.axpby_group(1.0, gs, momentum, vs, vs)
        if nesterov:
            us = [torch.empty_like(g) for g in gs]
            ops.axpby_group(1.0, gs, momentum, vs, us)
        ops.orthogonalize(
            us, steps=steps, coefficients=coef, eps=eps,
            scale=[rule._scale_of(p.data) for rule, p, _ in group],
            params=[p.data for _, p, _ in group], lr=lr, decay=decay)


def update_together(params):
    """``update`` of the parameters whose rule is exactly this one and has no
    hooks, all at once; the others are returned."""
    mine, rest = [], []
    for param in params:
        rule = param.update_rule
        if type(rule) is OrthogonalUpdateRule and rule.enabled and \
                not rule._pre_update_hooks and not rule._post_update_hooks:
            mine.append((rule, param))
        else:
            rest.append(param)
    for rule, param in mine:
        rule.prepare(param)
    if mine:
        apply_rules(mine)
    return rest
