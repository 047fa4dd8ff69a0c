"""The largest products in e4m3: more threads than one launch counts, in whole numbers, which are exact."""
import pytest
import torch

import ada_mla

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_more_tiles_than_a_launch(dtype):
    # 2^22 + 77 rows x 4096 outputs: 65 538 row tiles x 256 output tiles of 256 threads are more than 2^32 (34 GB of
    # outputs). Products of -1, 0 and 1 and their sums of 16 are exact in every type on the way.
    m, k, n = 2 ** 22 + 77, 16, 4096
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randint(-1, 2, (m, k), generator=gen, device="cuda").to(dtype)
    x[:, 0] = 1.0  # every row's scale is 1 / 448: its values stand at 448, 0 and -448
    w = torch.randint(-1, 2, (n, k), generator=gen, device="cuda").float()
    ws = torch.full((n // 128, 1), 2.0, device="cuda")
    y = ada_mla.mla_linear_fp8(x, w.to(torch.float8_e4m3fn), ws)
    step, wt = 2 ** 18, (w * 2).t().contiguous()
    # 448 (1 / 448) is 1 - 2^-24 in fp32 at worst: sums of up to 32 round to the same 16-bit value
    for at in range(0, m, step):
        assert torch.equal(y[at:at + step], (x[at:at + step].float() @ wt).to(dtype)), at
