"""What the operators for drafted tokens take and refuse, beside ``test_draft_cpu``."""
import pytest
import torch

from test_draft_cpu import BF16, _cache, _i32

from mesh_b200.ops.draft import draft_attention


def test_strides_of_dimensions_of_one_do_not_matter():
    """A single head, token or sequence has no neighbour for its stride to lead to: refused for want of a GPU alone."""
    c = _cache(B=1, H=1)
    x = torch.zeros(4096, dtype=BF16)
    for strides in ((777, 333, 111, 1), (64, 64, 64, 1), (0, 0, 0, 1)):
        q = x.as_strided((1, 1, 1, 64), strides)
        with pytest.raises(ValueError, match="GPU"):
            draft_attention(q, c, _i32(3), out=q)
    two = _cache(B=2, H=1)
    q = x.as_strided((2, 3, 1, 64), (1000, 200, 7, 1))
    with pytest.raises(ValueError, match="GPU"):
        draft_attention(q, two, _i32(3, 4), out=q.clone(memory_format=torch.preserve_format))
    with pytest.raises(ValueError, match="dense"):
        draft_attention(x.as_strided((2, 3, 2, 64), (1000, 200, 100, 1)), two, _i32(3, 4))
