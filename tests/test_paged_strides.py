"""Row strides that a C int would take for others are refused by the paged cache's Python calls, before anything is read. On the
CPU, with tensors that have no memory."""
import pytest
import torch

from hipinfer_amd import hipinfer as hi


def rows(M, width, stride, dtype):
    return torch.empty(0, dtype=dtype, device="meta").as_strided((M, width), (stride, 1))


@pytest.mark.parametrize("stride", [2**31, 2**32 + 512, 2**33 + 512])
def test_row_strides(stride):
    with pytest.raises(ValueError, match="2\\^31"):
        hi._rows_of("attn_paged", "q", rows(2, 512, stride, torch.float16), 2, 512)
    assert hi._rows_of("attn_paged", "q", rows(2, 512, 2**31 - 8, torch.float16), 2, 512) == 2**31 - 8
    assert hi._rows_of("attn_paged", "q", rows(1, 512, stride, torch.float16), 1, 512) == 512  # nothing is apart


@pytest.mark.parametrize("stride", [2**31, 2**32 + 4])
def test_table_strides(stride):
    pages = torch.empty(3, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="2\\^31"):
        hi._paged("attn_paged", pages, pages, rows(2, 4, stride, torch.int32), 1)
    assert hi._paged("attn_paged", pages, pages, rows(1, 4, stride, torch.int32), 1)[0][-2:] == (4, 4)
