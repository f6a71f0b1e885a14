"""Products with 4-bit weights where the kernel of few rows has the shortest ring of copies and the most sets of output rows a block."""
import pytest
import torch

from realhf_b200.ops import int4
from test_int4 import TYPES, check_linear, rows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group", [(9, 22016, 1024, 32), (16, 50257, 512, 32), (12, 4096, 11008, 32), (16, 33, 8192, 32), (13, 9600, 1056, 32), (16, 9600, 4096, 64), (8, 30000, 1056, 32),
                                         (16, 100, 32, 32)])
def test_few_rows_in_small_groups(dtype, M, N, K, group):
    g = torch.Generator().manual_seed(M + N + K)
    lin = int4.Int4Linear(rows(g, N, K, dtype=dtype, device="cuda") * K ** -0.5, group=group)
    check_linear(lin, rows(g, M, K, dtype=dtype, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group", [(17, 1, 32, 32), (20, 129, 96, 32), (64, 40, 64, 64), (100, 300, 32, 32), (128, 257, 160, 32), (129, 130, 192, 64), (257, 16, 128, 128)])
def test_many_rows_over_few_channels(dtype, M, N, K, group):
    g = torch.Generator().manual_seed(M + N + K)
    lin = int4.Int4Linear(rows(g, N, K, dtype=dtype, device="cuda") * K ** -0.5, rows(g, N, 1, dtype=dtype, device="cuda")[:, 0], group)
    check_linear(lin, rows(g, M, K, dtype=dtype, device="cuda"))
