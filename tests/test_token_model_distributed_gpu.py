"""An embedding's block under ``DistributedKFAC`` against one process on the
whole batch.  The two ranks are threads of one process that take turns: one
runs from collective to collective, everything it has queued is done before the
other goes on, and the arrays change hands on the host."""

import threading

import pytest
import torch
from torch import nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

RANKS = 2
SECONDS = 60


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')


class Exchange(object):
    """Where the ranks meet: all bring something, all get everything."""

    def __init__(self):
        self.turn = threading.Lock()
        self.meet = threading.Barrier(RANKS)
        self.brought = [None] * RANKS

    def all_of(self, rank, what):
        torch.cuda.synchronize()
        self.brought[rank] = what
        self.turn.release()
        try:
            self.meet.wait(SECONDS)
        finally:
            self.turn.acquire()
        got = list(self.brought)
        self.turn.release()
        try:
            self.meet.wait(SECONDS)
        finally:
            self.turn.acquire()
        return got


class Comm(object):

    def __init__(self, exchange, rank):
        self.exchange, self.rank, self.size = exchange, rank, RANKS

    @staticmethod
    def _copies(arrays):
        return [[a.clone() for a, _ in part] for part in arrays]

    def bcast_data(self, model):
        params = [p for _, p in sorted(model.namedparams())]
        got = self.exchange.all_of(self.rank, [p.data.clone() for p in params])
        for p, x in zip(params, got[0]):
            p.data.copy_(x)

    def reduce_scatter_v_arrays(self, arrays, stream=None):
        got = self.exchange.all_of(self.rank, self._copies(arrays))
        for k, (a, _) in enumerate(arrays[self.rank]):
            a.copy_(sum(g[self.rank][k] for g in got) / RANKS)
        torch.cuda.synchronize()

    def all_gather_v_arrays(self, arrays, stream=None):
        got = self.exchange.all_of(self.rank, self._copies(arrays))
        for owner, part in enumerate(arrays):
            for k, (a, _) in enumerate(part):
                a.copy_(got[owner][owner][k])
        torch.cuda.synchronize()


def make():
    import chainerkfac_b200 as ck
    torch.manual_seed(3)
    return nn.Sequential(
        ck.EmbedID(33, 14, ignore_label=-1, scale=1.5, device='cuda'),
        nn.Linear(14, 20, device='cuda'), nn.Tanh(),
        nn.Linear(20, 11, device='cuda'))


def lossfun(model):
    return lambda ids, t: F.cross_entropy(model(ids).flatten(0, -2),
                                          t.flatten())


def batches(steps):
    out = []
    for k in range(steps):
        g = torch.Generator(device='cuda')
        g.manual_seed(k)
        ids = torch.randint(33, (8, 6), device='cuda', generator=g)
        ids[:, 5:] = -1
        out.append((ids, torch.randint(11, (8, 6), device='cuda',
                                       generator=g)))
    return out


def run_ranks(work):
    exchange, errors, got = Exchange(), [], [None] * RANKS

    def run(rank):
        exchange.turn.acquire()
        try:
            got[rank] = work(Comm(exchange, rank))
            torch.cuda.synchronize()
        except BaseException as e:           # shown below
            errors.append(e)
            exchange.meet.abort()
        finally:
            exchange.turn.release()
    threads = [threading.Thread(target=run, args=(r,)) for r in range(RANKS)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    real = [e for e in errors if not isinstance(e, threading.BrokenBarrierError)]
    if errors:
        raise (real or errors)[0]
    return got


@pytest.mark.parametrize('pic,early,own,decay,acc,loss_scale', [
    (True, False, 'reference', 0.9, 1, None),
    (False, False, 'reference', 0.9, 1, None),
    (True, True, 'balanced', 0.9, 1, None),
    (False, True, 'reference', 1.0, 1, None),
    (True, False, 'balanced', 0.9, 2, None),
    (True, False, 'reference', 0.9, 1, 64.0),
    (False, False, 'balanced', 0.9, 1, 64.0)])
def test_two_ranks_are_one_process(pic, early, own, decay, acc, loss_scale):
    """Factors agree to 1e-4 and updates to 1e-3, what the framework holds its
    blocks to."""
    import chainerkfac_b200 as ck
    from chainerkfac_b200.optimizers import fisher_blocks as FB
    steps = 3
    data = batches(steps * acc)
    kw = dict(lr=0.05, momentum=0.9, cov_ema_decay=decay, damping=1e-2,
              acc_iters=acc, loss_scale=loss_scale)

    def work(comm):
        torch.cuda.set_device(0)
        model = make()
        opt = ck.DistributedKFAC(comm, only_pic_update_weight=pic,
                                 communicate_after_forward=early,
                                 ownership=own, **kw).setup(model)
        part = slice(4 * comm.rank, 4 * comm.rank + 4)
        opt.is_changed(opt.target)           # (weights are alike already)
        for ids, t in data:
            opt.update(lossfun(model), ids[part], t[part])
        assert opt.t == steps
        return model, opt
    got = run_ranks(work)
    one = make()
    start = one[0].weight.detach().clone()
    ref = ck.KFAC(**kw).setup(one)
    for ids, t in data:
        ref.update(lossfun(one), ids, t)
    for a, b in zip(got[0][0].parameters(), got[1][0].parameters()):
        assert torch.equal(a, b)
    owned = 0
    for model, opt in got:
        for i in opt.local_indices:
            fb, same = opt.fblocks[i], ref.fblocks[i]
            for x, y in zip(fb.cov_emas, same.cov_emas):
                assert float((x - y).norm()) <= 1e-4 * float(y.norm())
            owned += isinstance(fb, FB.FisherBlockEmbedID)
        step, want = model[0].weight.detach() - start, one[0].weight - start
        assert float((step - want).norm()) <= 1e-3 * float(want.norm())
        for x, y in zip(model.parameters(), one.parameters()):
            assert float((x - y).norm()) <= 1e-3 * float(y.norm())
    assert owned == 1
