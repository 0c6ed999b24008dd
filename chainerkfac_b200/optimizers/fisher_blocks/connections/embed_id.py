"""Block of a token embedding: the block of a fully connected layer without
bias (``chainerkfac/optimizers/fisher_blocks/connections/linear.py``) on rows
that are ``scale`` at the token's place and zero elsewhere.

The input factor A = scale^2 diag(counts) / n is kept as its diagonal, beside
it its mean, which is what the damping's pi needs of its trace:
``covs`` / ``cov_emas`` are [A (vocab,), G (width, width), mean (1, 1)], and
``invs`` those of [mean, G]: what the inverse of the mean was damped with is
added to A's diagonal in the update."""

import torch

from chainerkfac_b200 import ops
from chainerkfac_b200.optimizers.fisher_blocks.connection import \
    FisherBlockConnection


class EmbedIDFunction(object):
    """Marks a call of an embedding in the hook protocol."""


class FisherBlockEmbedID(FisherBlockConnection):

    def __init__(self, *args, **kwargs):
        self._mean = None
        super(FisherBlockEmbedID, self).__init__(*args, **kwargs)

    @property
    def funcclass(self):
        return EmbedIDFunction

    def dims(self):
        return self.link.W.shape

    # -- factors ----------------------------------------------------------
    def forward_postprocess(self, func, in_data):
        super(FisherBlockEmbedID, self).forward_postprocess(func, in_data)
        if not self.deferred:
            self.covs = [self._A, self._G, self._mean]

    def backward_preprocess(self, func, in_data, out_grad_data):
        super(FisherBlockEmbedID, self).backward_preprocess(
            func, in_data, out_grad_data)
        if not self.deferred:
            self.covs = [self._A, self._G, self._mean]

    def flush_items(self, forward_only=False):
        pend, items = getattr(self, '_pending_A', None), []
        if pend is not None:
            self._A = self.compute_A(pend)
            self._pending_A = None
        had_G = getattr(self, '_pending_G', None) is not None
        items = super(FisherBlockEmbedID, self).flush_items(forward_only)
        if pend is not None or had_G:
            self.covs = [self._A, self._G, self._mean]
        return items

    def compute_A(self, in_data):
        ids = in_data[0].contiguous()
        vocab, link = self.link.W.shape[0], self.link
        if ids.numel() == 0:
            raise ValueError('%s: a batch with no tokens has no factors'
                             % self.linkname)
        if self._A is None or self._A.device != ids.device:
            self._A = torch.empty(vocab, dtype=torch.float32,
                                  device=ids.device)
            self._mean = torch.empty((1, 1), dtype=torch.float32,
                                     device=ids.device)
        return ops.token_counts(ids, vocab, link.ignore_label,
                                alpha=link.scale ** 2 / ids.numel(),
                                out=self._A, mean=self._mean)

    def compute_G(self, in_data, out_grad_data):
        gy = self._rows(out_grad_data[0])
        s = self.gy_scale(gy.shape[0])
        out = self.factor_buffer(1, gy.shape[1], gy.device)
        return ops.factor_dense(gy, False, alpha=s * s / gy.shape[0], out=out)

    def item_G(self, in_data, out_grad_data):
        gy = self._rows(out_grad_data[0])
        s = self.gy_scale(gy.shape[0])
        self._G = self.factor_buffer(1, gy.shape[1], gy.device)
        self._keep_gy = gy
        return ops.dense_item(gy, False, s * s / gy.shape[0], 0.0, self._G)

    @staticmethod
    def _rows(gy):
        return gy.reshape(-1, gy.shape[-1]).contiguous()

    # -- inverses ---------------------------------------------------------
    def plan_factors(self):
        return [] if self.cov_emas is None else \
            [self.cov_emas[2], self.cov_emas[1]]

    def max_side(self):
        return int(self.covs[1].shape[0])

    def ensure_invs(self):
        if self.invs is None:
            self.invs = [torch.empty_like(f) for f in self.plan_factors()]
        return self.invs

    def update_invs(self):
        self.check_attr('cov_emas')
        self.ensure_invs()
        if self._plan is None:
            entries = self.plan_entries()
            self._plan = ops.InversePlan(
                self.plan_factors(), self.invs, [1, 0],
                [e[0] for e in entries], [e[1] for e in entries],
                [e[2] for e in entries])
        self._plan.run(self.damping, self._pi_type == 'tracenorm')
        self.set_diag_vals(self._plan.diag)

    def get_diagvals(self):
        if self._plan is None:
            self.update_invs()
        return [self.diag_val_forward.expand(self.cov_emas[0].shape[0]),
                self.diag_val_backward.expand(self.cov_emas[1].shape[0])]

    # -- update -----------------------------------------------------------
    def precondition(self, param=None, mom=None, lr=0.0, momentum=0.0):
        """kf = diag(1 / (A + damping)) grad G_inv into ``W.kfgrad``, and the
        momentum update of a weight that is given."""
        self.check_attr('invs')
        W = self.link.W
        kfW, _ = self.kfgrad_buffers()
        ops.precondition_embedding(
            self.invs[1], self.cov_emas[0], self._diag_src[0],
            W.grad.contiguous(), kfW, param, mom, lr, momentum)

    def update_kfgrads(self):
        self.precondition()

    # -- arrays moved by the collectives ----------------------------------
    def extract_for_reduce_scatter_v_after_forward(self):
        if self._communicate_after_forward:
            return [(self.covs[0], False), (self.covs[2], False)]
        return []

    def extract_for_reduce_scatter_v(self):
        arrays = self.extract_attr_from_params('grad')
        if not self._communicate_after_forward:
            arrays += [(self.covs[0], False), (self.covs[2], False)]
        arrays.append((self.cov_backward, True))
        return arrays
