"""How much of an adapter's first product reaches its second."""
import pytest
import torch

pytestmark = pytest.mark.gpu



@pytest.fixture(scope="module")
def ops():
    from ninfer_amd.kernels import load_ops
    return load_ops()


@pytest.mark.parametrize("rows,r,k", [(1, 16, 64), (16, 2, 72), (3, 7, 33), (1, 64, 64), (20, 12, 136), (40, 9, 65), (2048, 64, 64), (1700, 33, 40)])
def test_adapters_hand_on_all_bits_of_the_first_product(ops, rows, r, k):
    """Two numbers of h that differ in the last of their 24 bits, one taken from the other: every sum is a whole number that 32 bits
    hold, so that nothing may be lost."""
    n, g = 200, 1
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 2.0 ** 23, 2.0 ** 15, 2.0 ** 7, 1.0
    a = torch.zeros(2, r, k, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(2, n, r, dtype=torch.bfloat16, device="cuda")
    a[g, 0, :4], a[g, r - 1, :3] = 1.0, 1.0
    sign = torch.tensor([1.0, -1.0], device="cuda")[torch.arange(n, device="cuda") % 2].bfloat16()
    b[g, :, 0], b[g, :, r - 1] = sign, -sign
    scale, ranks = torch.ones(2, device="cuda"), torch.tensor([r, r], dtype=torch.int32, device="cuda")
    of = torch.full((rows,), g, dtype=torch.int32, device="cuda")
    out = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    ops.adapter_add(x, a, b, scale, ranks, (n,), of, out)
    assert torch.equal(out, sign.expand(rows, n))
