"""The CSR of a matrix of more than 2^26 rows and its transpose (64 work-items a row are over 2^32)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_transpose_of_very_many_rows(device):
    from gnnea.graph import DeviceCSR
    n = 2 ** 26 + 5
    row = torch.tensor([0, 0, 3, 2 ** 25 - 1, 2 ** 25, 2 ** 26 - 1, 2 ** 26, n - 1, n - 1])
    col = torch.tensor([1, 2, 0, 2, 1, 0, 2, 0, 1])
    adj = DeviceCSR.from_coo(row.to(device), col.to(device), None, n, 3)
    assert adj.row_ids().tolist() == row.tolist()
    t = adj.transpose()
    want = sorted(zip(col.tolist(), row.tolist()))
    assert t.nnz == len(row) and t.col.tolist() == [r for _, r in want]
    assert t.rowptr.tolist() == [0, 3, 6, 9]
