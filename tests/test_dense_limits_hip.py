"""More rows than one launch has threads for (2^32): norms, 8-bit rows and the rows that are padded."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_narrow_rows(device):
    """2^28 rows of one value are 2^32 threads.  Without eps the norm of a number is its sign."""
    from maloq_amd.dense import quantize_rows
    from maloq_amd.norm import rms_norm
    rows = 2 ** 28 + 37
    x = torch.randint(1, 100, (rows, 1), device=device, dtype=torch.int16).bfloat16()
    x[::3] *= -1
    w = torch.full((1,), 1.5, device=device, dtype=torch.bfloat16)
    assert torch.equal(rms_norm(x, w, 0.0), x.sign() * 1.5)
    q, scale = quantize_rows(x)
    assert torch.equal(q.view(torch.int8) < 0, x < 0) and torch.equal((scale * 448).bfloat16(), x[:, 0].abs())


def test_wide_rows(device):
    """A row of more than 1024 values is a workgroup's: 2^24 of them."""
    from maloq_amd.dense import quantize_rows
    rows, n = 2 ** 24 + 5, 1025
    x = torch.randn(1, n, device=device)
    q, scale = quantize_rows(x.expand(rows, n))
    one, s = quantize_rows(x)
    assert bool((scale == s).all())
    for at in (0, 2 ** 24 - 20, rows - 20, *range(0, rows - 20, 1234567)):
        assert bool((q[at:at + 20].view(torch.uint8) == one.view(torch.uint8)).all()), at


def test_padded_rows(device):
    """16 bytes of the result a thread."""
    from maloq_amd import _lib
    n, k, kp = 7, 1001, 1008
    rows = 2 ** 32 // (kp // 8) + 9
    if torch.cuda.mem_get_info(device)[0] < rows * kp * 2 + 2 ** 32:
        pytest.skip("needs 73 GB of free memory")
    x, w = (torch.randn(m, k, device=device).bfloat16() for m in (1, n))
    xp = torch.empty(rows, kp, device=device, dtype=torch.bfloat16)
    wp = torch.empty(n, kp, device=device, dtype=torch.bfloat16)
    for at in (0, rows // 2, rows - 20):
        xp[at:at + 20] = 1
    _lib.call("maloq_linear_pad", 1, x, 0, rows, w, k, n, k, xp, wp, _lib.stream_of(device))
    assert torch.equal(wp[:, :k], w) and not wp[:, k:].any()
    for at in (0, rows // 2, 2 ** 32 // (kp // 8) - 20, rows - 20, *range(0, rows - 20, 1234567)):
        assert bool((xp[at:at + 20, :k] == x).all()) and not xp[at:at + 20, k:].any(), at
    del xp
    torch.cuda.empty_cache()
