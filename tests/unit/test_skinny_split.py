"""Split-K of the decode projections: the split belongs to both sizes of a
weight, and one that does not divide K is refused."""

import pytest
import torch

from calfkit_amd import ops
from calfkit_amd.models.config import get_config
from calfkit_amd.models.llama import LlamaShard


def test_split_divides_each_projection():
    """o and down have the same rows and another K."""
    model = LlamaShard(get_config("smoke", layers=1), device="cpu")
    lw = model.layers[0]
    for w in (lw.wqkv, lw.wo, lw.wgateup, lw.wdown, lw.wo):
        sk = model._splitk_for(w, 8)
        assert sk == ops.choose_splitk(*w.shape, 8)
        assert w.shape[1] % (sk * 4 * 32) == 0


@pytest.mark.gpu
def test_uneven_split_is_refused():
    x = torch.zeros(8, 2816, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(1024, 2816, dtype=torch.bfloat16, device="cuda")
    work = torch.zeros(8 * 16 * 1024, device="cuda")
    with pytest.raises(RuntimeError):
        ops.skinny_gemm_slabs(x, w, work, 8)
    act = torch.zeros(8, 512, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        ops.skinny_gemm_silu(act, x, w, work, 8)
