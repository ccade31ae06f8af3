"""The serving operators where their inputs reach the ends of what the entries accept: zero points beyond four bits, scales that
lie far apart, rows whose squares vanish in 32 bits, empty extents, non-finite rows, the status word under capture."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from . import serving_reference as ref  # noqa: E402
from .test_serving_gpu import CACHE, E4M3, I8, BF16, F16, F32, _check_attention, _check_norm, _check_w4, _cuda, _gen, _paged, _w4_case, ops  # noqa: E402,F401


# ---- zero points ------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 5, 12, 40, 130])
@pytest.mark.parametrize("n,k,group", [(77, 1024, 128), (130, 1056, 32), (300, 2048, 32), (256, 1088, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, E4M3, I8])
def test_w4_zero_points_beyond_four_bits(ops, m, n, k, group, dtype):
    """0 .. 127 are exact: 16 is what formats that store a zero point less one in four bits decode to."""
    d, out = _w4_case(m, n, k, dtype, group, True, True, 1, F32, out_dtype=F32)
    d["zeros"] = torch.randint(0, 128, d["zeros"].shape, generator=_gen(m + n), dtype=torch.uint8)
    d["zeros"].view(-1)[::7] = 16
    d["zeros"].view(-1)[::11] = 127
    _check_w4(ops, d, out)


@pytest.mark.parametrize("m", [1, 12, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_every_zero_point_and_nibble(ops, m, dtype, group):
    """x one-hot and scales of 1: q - z comes back exactly (in f32) up to 127; a zero point above is NaN in its row and in no other."""
    n, k = 256, 512
    q = torch.randint(0, 256, (n, k // 2), generator=_gen(m), dtype=torch.uint8)
    zeros = torch.arange(n, dtype=torch.uint8)[:, None].repeat(1, k // group)
    zeros[:128, 0] = 127 - zeros[:128, 0]  # another zero point in one of the groups
    scales = torch.ones(n, k // group)
    w = ref.w4_weights(q, scales, zeros, group)
    for at in (0, 33, 300, k - m):
        x = torch.zeros(m, k, dtype=dtype)
        x[torch.arange(m), at + torch.arange(m)] = 1.0
        got = ops.w4_matmul(x.cuda(), q.cuda(), scales.cuda(), zeros=zeros.cuda(), group=group, out_dtype=F32).cpu()
        assert torch.equal(got[:, :128].double(), w[:128, at:at + m].t())
        assert torch.isnan(got[:, 128:]).all()
