"""The residual norm's 8-bit output on the borders of its rounding."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_encoder_ops import BF16, E4M3, F32, g  # noqa: E402, F401


@pytest.mark.parametrize("C", [1024, 1031])
@pytest.mark.parametrize("group", [0, 64, 7])
@pytest.mark.parametrize("top", [574.0, 1344.0, 451.0, 7.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quotients_midway_between_two_values_go_to_the_even_one(g, C, group, top, dtype):
    """Rows of +-1 without eps have a root of exactly 1, so that y is the weight. The weights are odd multiples of a 32nd of
    a power of two, which lie midway between two e4m3 values, times the scale. Where the scale is exact in fp32 (not
    451 / 448) so are the products and their quotients, and one rounding is right; elsewhere it is that of the fp32
    quotient, which a 64-bit quotient of fp32 numbers rounds to without error."""
    scale = top / 448.0
    ties = torch.arange(17, 32, 2).float() / 16
    quotients = torch.cat([ties * 2.0 ** e for e in range(-5, 8)] + [-ties * 4.0])
    quotients = quotients[quotients.abs() < 440]
    w = quotients.repeat(C // len(quotients) + 1)[:C].double() * scale
    w[::group or C] = top  # every group has the same largest value
    y = w.float()
    assert top == 451.0 or torch.equal(y.double(), w)
    x = torch.where(torch.arange(3 * C).view(3, C) % 3 == 1, -1.0, 1.0)
    out, s = g.add_rms_norm_device(x.to(dtype).cuda(), None, y.cuda(), eps=0.0, out_dtype=E4M3, group=group)
    assert torch.equal(s.cpu(), torch.full_like(s.cpu(), scale))
    want = (x.double() * y.double() / s.cpu()[0, 0].double()).float().to(E4M3)
    assert torch.equal(out.cpu().float(), want.float())
