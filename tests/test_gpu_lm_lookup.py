"""What the LM's token lookup leaves to the module itself, as before there was a lookup of the framework's own."""
import pytest
import torch
import torch.nn as nn

from hdcmamba_b200.lm import embed

pytestmark = pytest.mark.gpu


def table(**kw):
    torch.manual_seed(0)
    return nn.Embedding(20, 16, **kw).cuda()


IDS = [[3, 1, 3], [7, 0, 19]]


def test_modules_of_other_kinds():
    class Sum(nn.Module):
        def __init__(self):
            super().__init__()
            self.parts = nn.ModuleList([table(), table()])

        def forward(self, ids):
            return self.parts[0](ids) + self.parts[1](ids)

    ids = torch.tensor(IDS).cuda()
    m = Sum()
    assert torch.equal(embed(m, ids), m(ids))
    f = table().weight.detach()
    assert torch.equal(embed(lambda i: f[i], ids), f[ids])
