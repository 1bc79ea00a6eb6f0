"""CPU: what Context.dispatch refuses: the library reads sel as contiguous int32 on the context's GPU, whatever it is."""
import pytest
import torch

import loki_amd


class Bare(loki_amd.Context):
    """a context's checks without a GPU"""
    def __init__(self):
        self.torch, self.ctx, self._device = torch, None, 0


@pytest.mark.parametrize("sel", [torch.topk(torch.randn(4, 16), 2, dim=1).indices, torch.zeros((4, 2), dtype=torch.int32), torch.zeros(8, dtype=torch.int32)],
                         ids=["int64", "not on the GPU", "one row of no shape"])
def test_dispatch_refuses(sel):
    with pytest.raises(loki_amd.LokiError, match="dispatch: "):
        Bare().dispatch(sel, n_exp=16)
