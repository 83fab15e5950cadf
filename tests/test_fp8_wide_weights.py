"""linear_fp8 on weights so wide that the launch that quantises the rows itself does not hold them: the rows are then
quantised ahead, and the product is mm_fp8's."""
import pytest
import torch

from lockstep_amd import _lib as L

WIDEST = 64 * (2 ** 24 - 1)     # columns of 2^24 - 1 blocks of 64: HIP launches fewer than 2^32 threads, 256 a block


def test_workspace_where_one_launch_does_not_hold_the_columns():
    lib = L.load()
    assert lib.lsk_linear_fp8_workspace(1, WIDEST, 16) == 0
    assert lib.lsk_linear_fp8_workspace(16, WIDEST, 1024) == 0
    assert lib.lsk_linear_fp8_workspace(1, WIDEST + 1, 16) == 512
    assert lib.lsk_linear_fp8_workspace(16, WIDEST + 1, 1024) == 16 * 1024 + 512


@pytest.mark.gpu
def test_linear_past_the_widest_launch():
    from lockstep_amd import lockstep_fullstack as FS
    N, K = 2 ** 30 + 200, 16
    print("linear", 1, N, K, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((1, K), generator=g, device="cuda")
    w = torch.zeros((N, K), dtype=torch.uint8, device="cuda")
    w[-1000:] = torch.randint(0, 120, (1000, K), generator=g, device="cuda").to(torch.uint8)
    w[:1000] = torch.randint(0, 120, (1000, K), generator=g, device="cuda").to(torch.uint8)
    w = w.view(torch.float8_e4m3fn)
    ws = torch.rand(((N + 127) // 128, 1), generator=g, device="cuda")
    y = FS.linear_fp8(x, w, ws, out_dtype=torch.bfloat16)
    first, last = 1024, N // 128 * 128 - 1024            # (on the scales' blocks)
    assert torch.equal(y[:, :first], FS.linear_fp8(x, w[:first], ws[:first // 128], out_dtype=torch.bfloat16))
    assert torch.equal(y[:, last:], FS.linear_fp8(x, w[last:], ws[last // 128:], out_dtype=torch.bfloat16))
    assert (y[:, first:last] == 0).all()
