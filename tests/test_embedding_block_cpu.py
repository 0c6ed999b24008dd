"""Host side of the embedding's block: calls that it refuses."""

import pytest
import torch


@pytest.mark.parametrize('deferred', [True, False])
def test_an_empty_batch_has_no_factors(deferred):
    import chainerkfac_b200 as ck
    opt = ck.KFAC().setup(ck.EmbedID(7, 4))
    fb = opt.fblocks[0]
    fb.deferred = deferred
    ids = torch.zeros((3, 0), dtype=torch.int64)
    with pytest.raises(ValueError, match='no tokens'):
        fb.forward_postprocess(fb.funcclass(), (ids, fb.link.W.data))
        fb.flush_items()
    assert fb.covs is None
