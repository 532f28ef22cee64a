"""Under autocast, a Linear that keeps its input in 8 bits casts what an ordinary Linear casts, and refuses the rest."""
from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from stagehand_amd.act8 import linear_act8

pytestmark = pytest.mark.gpu


def test_types_that_autocast_leaves_alone_are_refused():
    x, w, b = torch.ones(4, 64, device="cuda"), torch.ones(8, 64, device="cuda"), torch.ones(8, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for args in ((x.double(), w.double()), (x.double(), w), (x, w.double()), (x, w, b.double()), (x.long(), w), (x, w.long()), (x, w, b.int()),
                     (x.bool(), w)):
            with pytest.raises(ValueError, match="type"):
                linear_act8(*args)
        for args in ((x, w), (x.half(), w, b), (x.bfloat16(), w.half(), b)):  # these are cast
            y = linear_act8(*args)
            assert y.dtype == torch.bfloat16 and torch.equal(y, F.linear(*args))
