"""The gradient of the learned relative position bias's weight: every pair counted once, whatever the sizes and strides; the rounding of a
32-bit sum no larger than its longest chain; infinities, NaN and large numbers in their own bucket, wherever in a strip of
diagonals they stand."""
import pytest
import torch

from serving_helpers import dev, gen, half_step, randn, serving_oracle, spread

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


SHAPES = [(1, 1, 0), (1, 700, 699), (700, 1, 0), (7, 5, 0), (64, 64, 0), (129, 257, 128), (255, 1031, -40), (530, 520, 0), (1025, 300, 5000), (520, 1100, 3),
          (2, 4099, 2048), (33, 2049, 0), (600, 7, -300), (16, 512, 0), (17, 505, 1)]
BUCKETS = [(32, 128, True), (32, 128, False), (8, 20, True), (64, 700, True), (2, 5, False), (5, 9, False), (256, 900, True)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("Tq,Tk,off", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wdtype", DTYPES)
def test_whole_numbers_are_exact(Tq, Tk, off, dtype, wdtype):
    """sums of whole numbers up to 4 stay below 2^24: exact in 32 bits, rounded once to the weight's type.  A pair left out or counted
    twice shows, in every layout"""
    i = SHAPES.index((Tq, Tk, off))
    nb, md, both = BUCKETS[(i + DTYPES.index(dtype)) % len(BUCKETS)]
    H = 1 + i % 4
    dy = torch.randint(1, 5, (1, H, Tq, Tk), generator=gen(640 + i)).to(dtype)
    layouts = {"plain": dev(dy), "gaps": dev(spread(dy, (2, 3))), "shifted": dev(torch.cat([dy[..., :1], dy], -1))[..., 1:],
               "heads inside": dev(dy.transpose(1, 2).contiguous()).transpose(1, 2)}
    # the values up to 4 x 307500 pairs: fp16 ends at 65504, where the rounding is to infinity
    want = serving_oracle.relative_bias_grad(dy, nb, md, both, off)[0].float().to(wdtype)
    for name, x in layouts.items():
        got = _grad(x, nb, md, both, off, wdtype).cpu()
        assert torch.equal(got, want), (name, (got.double() - want.double()).abs().max())


@pytest.mark.parametrize("Tq,Tk,off", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rounding_of_the_sums(Tq, Tk, off, dtype):
    """The chain of 32-bit additions: at most `chunk` rows of a diagonal in a lane's register, one neighbour's, one rounding of the 64-bit
    sum; then a lane's share of the tasks (every 256th in each of four sums, the rest in one), two joins of the four and six of
    the lanes; one rounding.  chunk is the longest of 256 .. 16 that leaves 8 wavefronts to a compute unit."""
    i = SHAPES.index((Tq, Tk, off))
    nb, md, both = BUCKETS[(i + 3 * DTYPES.index(dtype)) % len(BUCKETS)]
    H = 1 + i % 4
    dy = randn(gen(660 + i), 1, H, Tq, Tk, dtype=dtype, shift=0.3)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for chunk in (256, 128, 64, 32, 16):
        tasks = -(-Tq // chunk) * -(-(Tk + chunk - 8) // 512)
        if tasks * H >= 8 * cus:
            break
    depth = chunk + 2 + tasks // 256 + 4 + 8
    ref, mag = serving_oracle.relative_bias_grad(dy, nb, md, both, off)
    got = _grad(dev(dy), nb, md, both, off).cpu().double()
    tol = depth * 2.0**-24 * mag
    assert ((got - ref).abs() <= tol + half_step(torch.float32) * (ref.abs() + tol)).all(), ((got - ref).abs() / tol.clamp(min=1e-30)).max()
