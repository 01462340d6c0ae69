"""Page tables that are parts of larger ones: the rows of a batch lie further apart than a row is long."""
import pytest
import torch

from tests import attention_reference as att
from tests.test_gpu_lm_attention import KINDS, filled, normal, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("head", [64, 60])
def test_decode_a_table_with_a_stride(gpu, dtype, kind, head):
    """By whole accesses and by the kernel for any head; one row for all sequences, too."""
    from matrix_b200 import lm

    lengths, page, pages = [70, 33, 1, 80], 16, 8
    cache, k, v = filled(lm, pages, page, 2, head, kind)
    table = tables(lengths, page, pages)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    q = normal(len(lengths), 6, head, dtype=dtype)
    wide = torch.cat([torch.full_like(table, 7), table, torch.full_like(table, -1)], 1).cuda()[:, table.shape[1]:2 * table.shape[1]]
    assert wide.stride(0) == 3 * wide.shape[1]
    want, bound = att.decode(q.double(), k, v, table, lengths, head ** -0.5, dtype)
    att.assert_close(lm.decode_attention(q.cuda(), cache, wide, n), want, bound)
    one = table[3:].expand(4, -1)
    want, bound = att.decode(q.double(), k, v, one, lengths, head ** -0.5, dtype)
    shared = table[3:].cuda().expand(4, -1)
    assert shared.stride(0) == 0
    att.assert_close(lm.decode_attention(q.cuda(), cache, shared, n), want, bound)
