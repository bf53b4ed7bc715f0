"""Products with 4-bit weights against the definition in 64 bits."""
import math

import pytest
import torch

from dtas_amd import _lib, ops
from gpu_util import Guarded

pytestmark = pytest.mark.gpu


def make(M, N, K, group, seed, offset=0):
    """Inputs on the host; on the device their data lies `offset` elements behind an aligned address."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).half()
    x[:, ::97] *= 8
    words = torch.randint(-2 ** 31, 2 ** 31, (N, K // 8), generator=g, dtype=torch.int64).to(torch.int32)
    scale = ((0.25 + torch.rand(N, K // group, generator=g)) / (2 * math.sqrt(K))).half()
    bias, res1, res2 = (torch.randn(*s, generator=g).half() for s in ((N,), (M, N), (M, N)))

    def there(t):
        raw = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        raw[offset:] = t.flatten().cuda()
        return raw[offset:].view(t.shape)

    return [x, words, scale, bias, res1, res2], [there(t) for t in (x, words, scale, bias, res1, res2)]


def weights(words, scale):
    N, K = words.shape[0], words.shape[1] * 8
    nibbles = (words[:, :, None].long() >> torch.arange(0, 32, 4)) & 15
    return (nibbles.double() - 7).view(N, scale.shape[1], -1) * scale.double()[:, :, None], K


def expected(host, epilogue, bias=True):
    """The value, and how far an answer may be from it.

    A group's products are exact and its sum has up to 128 of them, sums of groups are joined in any order by chains of up to K / 32 + 64
    additions in all: every rounding is 2^-24 of at most the sum of the magnitudes.  bias and residuals add three roundings
    of 2^-24, GELU (slope below 1.13) the error of its erfc, 2^-20 of the value with its products, and storing half a step: 2^-11 in fp16 (2^-25 below
    its normal range)."""
    x, words, scale, b, res1, res2 = host
    w, K = weights(words, scale)
    w = w.reshape(w.shape[0], K)
    y = x.double() @ w.t()
    slack = (K / 32 + 192) * 2.0 ** -24 * (x.double().abs() @ w.abs().t())
    if bias:
        y = y + b.double()
        slack = slack + 2.0 ** -24 * y.abs()
    if epilogue in (1, 2):
        y = y + res1.double() + res2.double()
        slack = slack + 2.0 ** -23 * (y.abs() + res1.double().abs() + res2.double().abs())
    if epilogue == 3:
        slack = 1.13 * slack
        y = y * 0.5 * torch.special.erfc(-y * math.sqrt(0.5))
        slack = slack + 2.0 ** -20 * y.abs() + 2.0 ** -30
    half = 2.0 ** -24 if epilogue == 2 else 2.0 ** -11
    return y, slack + half * (y.abs() + slack) + 2.0 ** -25


def check(M, N, K, group, epilogue, offset=0, bias=True, seed=0):
    host, device = make(M, N, K, group, seed + 7 * M + N + K, offset)
    x, words, scale, b, res1, res2 = device
    out = Guarded((M, N), torch.float32 if epilogue == 2 else torch.float16)
    two = epilogue in (1, 2)
    ops.gemv_q4(x, words, scale, b if bias else None, out.t, epilogue=epilogue, res1=res1 if two else None, res2=res2 if two else None)
    got = torch.from_numpy(out.check()).double()
    want, tolerance = expected(host, epilogue, bias)
    off = (got - want).abs() - tolerance
    assert bool((off <= 0).all()), (off.max().item(), (off > 0).sum().item())
    return out.t


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 64, 256), (1, 257, 2560), (1, 4096, 4096), (1, 100, 11008), (2, 33, 384), (3, 7, 128), (4, 300, 1024),
                                   (5, 511, 640), (8, 65, 2560), (13, 130, 4096), (16, 48, 896), (17, 2560, 256), (31, 17, 1280), (33, 200, 2560),
                                   (64, 129, 1152), (64, 2560, 10240), (65, 40, 512), (130, 70, 256)])
def test_sizes(M, N, K, group):
    check(M, N, K, group, 0)


@pytest.mark.parametrize("epilogue", [0, 2, 3])
@pytest.mark.parametrize("M,N,K,group", [(7, 8230, 320, 32), (16, 8193, 128, 128), (33, 4200, 192, 64), (64, 4130, 96, 32), (5, 8300, 1280, 128)])
def test_more_columns_than_one_round_of_narrow_blocks(M, N, K, group, epilogue):
    check(M, N, K, group, epilogue)


def test_many_rows_of_a_long_k():
    # the parts of all rows together are more than the workspace is asked for at once: several launches
    M, N, K, group = 4100, 8192, 5120, 32
    host, dev = make(M, N, K, group, 1)
    y = torch.empty(M, N, dtype=torch.float16, device="cuda")
    ops.gemv_q4(*dev[:4], y, _lib.EPI_BIAS_ADD2, *dev[4:])
    for rows in ([0, 31, 32, 1023, 2015, 2016, 2047, 2048, 2049], [4063, 4064, 4095, 4096, 4099]):
        value, slack = expected([host[0][rows], *host[1:4], host[4][rows], host[5][rows]], _lib.EPI_BIAS_ADD2)
        assert bool(((y[rows].cpu().double() - value).abs() <= slack).all())
    assert bool(torch.isfinite(y).all())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 4, 5, 16, 17, 64])
def test_small_products_beside_a_large_row_element(M, group):
    # x is one number of 1024 per group, which meets the weight 0, and whole numbers of 2^-10 up to 31: every product and every sum is a
    # whole number of 2^-10 below 2^24 of them (31 * 8 * 640 < 2^18), which fp32 holds: the sum is the exact one in any order
    N, K = 48, 640
    g = torch.Generator().manual_seed(M)
    nibbles = torch.randint(0, 16, (N, K), generator=g)
    x = torch.randint(-31, 32, (M, K), generator=g).double() / 1024
    x[:, 5::group] = 1024
    nibbles[:, 5::group] = 7
    words = (nibbles.view(N, K // 8, 8) << (4 * torch.arange(8))).sum(-1)
    words = (words - (words >> 31 << 32)).to(torch.int32)
    y = torch.empty(M, N, device="cuda")
    zero, one = torch.zeros(M, N, dtype=torch.float16, device="cuda"), torch.ones(N, K // group, dtype=torch.float16, device="cuda")
    ops.gemv_q4(x.half().cuda(), words.cuda(), one, None, y, _lib.EPI_BIAS_ADD2_CAST_F32, zero, zero)
    assert torch.equal(y.cpu().double(), x @ (nibbles - 7).double().T)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("M,N,K", [(1, 40, 65536), (4, 33, 20480), (3, 5000, 16384), (12, 50, 32768), (40, 70, 49152)])
def test_long_k(M, N, K, group):
    # K shared by workgroups because the LDS does not hold its scales, or x
    check(M, N, K, group, 0)


@pytest.mark.parametrize("epilogue", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", [(1, 515, 2560), (2, 96, 512), (7, 100, 640), (24, 333, 1024), (50, 64, 2560)])
def test_epilogues(M, N, K, epilogue):
    check(M, N, K, 32, epilogue)
    check(M, N, K, 128, epilogue, bias=False)


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("M", [1, 6, 20])
def test_data_off_every_boundary(M, offset):
    check(M, 70, 512, 32, 0, offset=offset)


@pytest.mark.parametrize("M", [1, 2, 5, 16, 40, 64])
@pytest.mark.parametrize("group", [32, 128])
def test_whole_numbers_come_out_exactly(M, group):
    # x of -3 .. 3 and scales 1 / 64: every sum is a multiple of 1 / 64 below 2^18, and what fits fp32 has no rounding at all
    N, K = 75, 1280
    host, _ = make(M, N, K, group, 5)
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-3, 4, (M, K), generator=g).half()
    scale = torch.full_like(host[2], 1 / 64)
    w, _ = weights(host[1], scale)
    y, zero = torch.empty(M, N, device="cuda"), torch.zeros(M, N, device="cuda", dtype=torch.float16)
    ops.gemv_q4(x.cuda(), host[1].cuda(), scale.cuda(), None, y, epilogue=_lib.EPI_BIAS_ADD2_CAST_F32, res1=zero, res2=zero)
    assert torch.equal(y.cpu().double(), x.double() @ w.reshape(N, K).t())


def test_every_nibble_in_every_place():
    # one-hot x: y[k, n] is the weight itself, for each of the eight places of a word and each of the sixteen values
    N, K = 16, 128
    words = torch.tensor([[sum(((n + j + i) % 16) << (4 * i) for i in range(8)) for j in range(K // 8)] for n in range(N)], dtype=torch.int64)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    scale = torch.ones(N, 1).half() * 0.5
    w, _ = weights(words, scale)
    for rows in (1, 3, 64, 128):
        x = torch.eye(K).half()
        y = torch.cat([torch.empty(0, N)] + [_product(x[at:at + rows], words, scale, N) for at in range(0, K, rows)])
        assert torch.equal(y.double(), w.reshape(N, K).t())


def _product(x, words, scale, N):
    y = torch.empty(x.shape[0], N, device="cuda", dtype=torch.float16)
    ops.gemv_q4(x.cuda(), words.cuda(), scale.cuda(), None, y)
    return y.cpu().float()


def test_infinities_stay_in_their_rows():
    host, (x, words, scale, b, _, _) = make(20, 48, 256, 32, 1)
    x[3, 5], x[11, 100] = float("inf"), float("nan")
    y = torch.empty(20, 48, device="cuda", dtype=torch.float16)
    ops.gemv_q4(x, words, scale, b, y)
    fine = [m for m in range(20) if m not in (3, 11)]
    assert bool(torch.isfinite(y[fine]).all()) and not bool(torch.isfinite(y[3]).any()) and bool(torch.isnan(y[11]).all())
    want, tolerance = expected(host, 0)
    assert bool(((y.cpu().double() - want).abs() <= tolerance)[fine].all())


def test_empty_k_is_the_bias():
    y = torch.full((3, 8), 5.0, device="cuda", dtype=torch.float16)
    bias = torch.arange(8, device="cuda").half()
    ops.gemv_q4(torch.empty(3, 0, device="cuda", dtype=torch.float16), torch.empty(8, 0, device="cuda", dtype=torch.int32),
                torch.empty(8, 0, device="cuda", dtype=torch.float16), bias, y)
    assert torch.equal(y, bias.expand(3, 8))


def test_refusals():
    h = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.float16)
    w = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)
    for args, why in (((h(2, 64), w(8, 8), h(8, 3), None, h(2, 8)), "groups of"), ((h(2, 64), w(8, 8), h(8, 4), None, h(2, 8)), "groups of"),
                      ((h(2, 64), h(8, 8), h(8, 2), None, h(2, 8)), "32-bit words"), ((h(2, 32), w(8, 8), h(8, 2), None, h(2, 8)), "inner extents"),
                      ((h(2, 64), w(8, 8), h(8, 2), h(7), h(2, 8)), "shape mismatch"), ((h(2, 64), w(8, 8), h(8, 2), None, h(3, 8)), "shape mismatch"),
                      ((h(2, 64), w(8, 8), h(8, 2), None, h(2, 8).float()), "expects fp16"), ((h(64, 2).t(), w(8, 8), h(8, 2), None, h(2, 8)), "compact")):
        with pytest.raises(ValueError, match=why):
            ops.gemv_q4(*args)
    with pytest.raises(_lib.DtasError, match="residuals"):
        ops.gemv_q4(h(2, 64), w(8, 8), h(8, 2), None, h(2, 8), epilogue=1)
