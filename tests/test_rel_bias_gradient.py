"""The gradient of the learned relative position bias's weight: infinities, NaN and large numbers stay in their bucket, wherever in a
strip of diagonals they stand."""
import pytest
import torch

from serving_helpers import gen, serving_oracle

pytestmark = pytest.mark.gpu

NB, MD = 32, 128


def _grad(dy, nb=NB, md=MD, both=True, off=0, wdtype=torch.float32):
    from rgd_triton_amd import relative_position_bias_fn

    H, Tq, Tk = dy.shape[1:]
    w = torch.zeros(nb, H, device="cuda", dtype=wdtype, requires_grad=True)
    return torch.autograd.grad(relative_position_bias_fn(w, Tq, Tk, max_distance=md, bidirectional=both, q_offset=off, dtype=dy.dtype), w, dy)[0]


# a strip is 512 columns and the 7 diagonals beside it; its last seven are kept by one lane alone.  (row, column): the ends of strips
# in tasks of 16 rows, in their first, second and last rows, and the matrix's corners
SPOTS = [(800, j) for j in range(494, 514)] + [(815, j) for j in range(510, 528)] + [(807, 510), (808, 511), (809, 512), (0, 0), (0, 1023), (1023, 0), (1023, 1023),
                                                                                     (0, 503), (0, 504), (0, 511), (16, 1015), (16, 1016), (31, 503), (500, 500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinities_stay_in_their_bucket(value, dtype):
    H, T = 2, 1024
    # small whole numbers: every finite sum is exact in 32 bits, whatever its order (1024 x 1024 x 4 = 2^22)
    dy = torch.randint(-4, 5, (1, H, T, T), generator=gen(600)).to(dtype).cuda()
    finite = _grad(dy)
    for i, j in SPOTS:
        bad = dy.clone()
        bad[0, 0, i, j] = value
        dw = _grad(bad)
        own = serving_oracle.bucket_of(j - i, NB, MD, True)
        hit = dw[own, 0].item()
        assert hit != hit if value != value else hit == value, (i, j, hit)
        rest = torch.ones(NB, H, dtype=torch.bool)
        rest[own, 0] = False
        assert torch.equal(dw.cpu()[rest], finite.cpu()[rest]), (i, j, dw[:, 0].tolist())


@pytest.mark.parametrize("value", [3e38, 1e30, 2.0**60])
def test_large_numbers_stay_in_their_bucket(value):
    """two large numbers on one diagonal, in one task or in two: their own sum is theirs alone (infinite where 32 bits end), the other
    buckets' whole numbers are exact beside them"""
    T = 1024
    dy = torch.randint(-4, 5, (1, 1, T, T), generator=gen(601)).float().cuda()
    finite = _grad(dy).cpu()
    for i, j in ((800, 503), (800, 504), (808, 509), (3, 300), (200, 190), (1000, 1001)):
        big = dy.clone()
        big[0, 0, i, j] = big[0, 0, i + 1, j + 1] = value
        dw = _grad(big).cpu()
        own = serving_oracle.bucket_of(j - i, NB, MD, True)
        # the whole numbers of the bucket vanish beside the two: all below 2^22, half a step of the smallest sum is 2^37
        assert dw[own, 0].item() == (torch.tensor(value) + torch.tensor(value)).item()
        rest = torch.arange(NB) != own
        assert torch.equal(dw[rest], finite[rest]), (i, j, dw[:, 0].tolist())


def test_many_ranges_in_a_strip():
    """256 buckets, so that every lane places several beginnings; whole numbers, compared with the sums along the diagonals"""
    for both, off, Tq, Tk in ((True, 0, 700, 900), (False, 300, 300, 700), (True, -1000, 40, 2100)):
        dy = torch.randint(-4, 5, (1, 3, Tq, Tk), generator=gen(602)).float()
        want, _ = serving_oracle.relative_bias_grad(dy, 256, 900, both, off)
        assert torch.equal(_grad(dy.cuda(), 256, 900, both, off).cpu().double(), want)
