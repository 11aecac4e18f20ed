"""The layer products at the edges of what they promise: how often a 16-bit result is not the nearest number, the largest
numbers of rows, features and groups, the longest depths and lines, one bias for all groups, results in the place of an operand."""
import pytest
import torch

from clblast_amd import api
from tests import layer_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_kept():
    """The largest of these tests hold 100 GB: what torch keeps of it goes back after each"""
    yield
    torch.cuda.empty_cache()


def nearest(value, dtype):
    """A 64-bit value rounded once. (The way over 32 bits rounds twice: it only matters within 2^-24 of a border, far less than the
    errors that are counted here.)"""
    return value.to(dtype)


@pytest.mark.parametrize("kind,low", (("gelu", -4.0), ("silu", -4.0), ("gelu_tanh", -2.0)))
def test_activations_are_nearly_always_rounded_to_nearest(gpu, kind, low):
    """act(z) on the negative side, where its accuracy is that of its tail, for 16-bit results of half a million different z.
    Off by e relative to its value, a result is rounded the wrong way where a border between two numbers lies within e of it: of
    a value in [2^q, 2^(q + 1)) the borders are 2^(q - 10) apart in fp16 and 2^(q - 7) in bf16, so that is a share of at most
    2 e 2^(q + 1) / 2^(q - 10) = 4096 e, or 512 e. e is 2^-20 at most: fit of Phi 2^-23.5, its evaluation and the hardware's
    exponential and reciprocal a few times 2^-24, the rounded argument of the exponential, at most 11.6 (gelu at -4: z^2 log2(e) / 2),
    3 (gelu_tanh at -2, of three roundings: 2u log2(e) is 5.4) or 5.8 (silu), times 2^-24 and less than that again for the rounded
    log2(e): in all below 16 of 2^-24. Five standard deviations of a count are added."""
    assert ref.FUNCTION[torch.float16] >= 2.0 ** -20
    g = torch.Generator().manual_seed(8)
    z = torch.arange(1, 1 << 14, dtype=torch.int32).to(torch.int16).view(torch.float16)
    z = -z[(z > 0.04) & (z <= -low)].float()
    n = z.numel() // 8 * 8
    z = z[:n].to("cuda:0")
    for dtype, share in ((torch.float16, 4096 * 2.0 ** -20), (torch.bfloat16, 512 * 2.0 ** -20)):
        one = torch.ones(1, 1, dtype=dtype, device="cuda:0")
        wrong = count = 0
        rows = z.to(dtype).unique()
        n = rows.numel()
        for alpha in (0.5 + 0.5 * torch.rand(64 if dtype == torch.float16 else 512, generator=g)).tolist():
            alpha = float(torch.tensor(alpha))
            c = torch.zeros(1, n, dtype=dtype, device="cuda:0")
            api.gemmEpilogue(None, 1, n, 1, one, rows, c, 1, n, n, alpha=alpha, activation=kind)
            exact = ref.act((rows.float() * alpha).double(), kind)  # (alpha times a value is rounded once to 32 bits, here as there)
            wrong += int((c[0] != nearest(exact, dtype)).sum())
            count += n
        most = share * count
        print("%s %s: %d of %d not rounded to nearest, at most %.0f expected" % (kind, dtype, wrong, count, most))
        assert wrong <= most + 5 * most ** 0.5 + 1, (kind, dtype, wrong, count, most)


def test_more_tiles_than_one_grid_holds(gpu):
    """2^30 rows of one feature are 2^24 tiles of 64 rows, or 2^23 of 128, in 2^32 threads. A depth of one, so that every value is a
    product alone: rounded once to fp16, by the product's fp32 sum exactly as by torch's."""
    m = (1 << 30) + 77
    g = torch.Generator(device="cuda:0").manual_seed(9)
    a = torch.randn(m, 2, generator=g, device="cuda:0", dtype=torch.float16)  # (rows at dwords: nothing is copied)
    b = torch.tensor([[1.25]], device="cuda:0", dtype=torch.float16)
    for variant in (0, 4, 6, 1):
        api.override_parameters(0, "Xlayer", 16, {"TILE_VARIANT": variant, "SPLIT_K": 0})
        try:
            c = torch.full((m + 3, 1), 7.0, device="cuda:0", dtype=torch.float16)
            api.gemmEpilogue(None, m, 1, 1, a, b, c, 2, 1, 1)
            torch.cuda.synchronize()
        finally:
            api.override_parameters(0, "Xlayer", 16, {"TILE_VARIANT": 0, "SPLIT_K": 0})
        assert torch.equal(c[:m, 0], a[:, 0] * b[0, 0]), variant
        assert bool((c[m:] == 7.0).all()), variant
        del c


def test_more_copied_lines_than_one_grid_holds(gpu):
    """2^30 rows of 17 elements, every second of which starts between dwords: four threads copy one"""
    m, k = (1 << 30) + 5, 17
    a = torch.empty(m * k, device="cuda:0", dtype=torch.float16)  # 36.5 GB
    part = torch.randn(1 << 20, k, generator=torch.Generator(device="cuda:0").manual_seed(10), device="cuda:0").round().half()
    rows = a.view(m, k)
    for at in range(0, m, 1 << 20):
        rows[at:at + (1 << 20)] = part[:min(1 << 20, m - at)]
    b = torch.ones(1, k, device="cuda:0", dtype=torch.float16)
    c = torch.full((m + 3, 1), 7.0, device="cuda:0", dtype=torch.float16)
    api.gemmEpilogue(None, m, 1, k, a, b, c, k, k, 1, b_transp=True)
    torch.cuda.synchronize()
    want = part.float().sum(1).half()  # (whole numbers: exact in any order)
    for at in range(0, m, 1 << 20):
        count = min(1 << 20, m - at)
        assert torch.equal(c[at:at + count, 0], want[:count]), at
    assert bool((c[m:] == 7.0).all())


def test_more_columns_to_add_up_than_one_grid_holds(gpu):
    """The sums of 2^30 features: 2^24 work-groups of 256 threads"""
    n = (1 << 30) + 70
    y = torch.randn(2, n, generator=torch.Generator(device="cuda:0").manual_seed(11), device="cuda:0", dtype=torch.float16)
    sums = torch.full((n + 3,), 7.0, device="cuda:0", dtype=torch.float16)
    api.activationGradient(None, 2, n, y, None, None, n, 0, 0, bias_gradient=sums)
    torch.cuda.synchronize()
    assert torch.equal(sums[:n], y[0] + y[1])  # (two values: one rounding)
    assert bool((sums[n:] == 7.0).all())


def test_the_most_rows_of_a_narrow_matrix(gpu):
    m = (1 << 31) - 1024
    y = torch.randn(m, generator=torch.Generator(device="cuda:0").manual_seed(12), device="cuda:0", dtype=torch.float16).sign_()
    y[5], y[-1] = 0.0, 0.0
    c = torch.full((m + 3,), 7.0, device="cuda:0", dtype=torch.float16)
    sums = torch.full((3,), 7.0, device="cuda:0", dtype=torch.float16)
    api.activationGradient(None, m, 1, y, y, c, 1, 1, 1, "relu", bias_gradient=sums)
    torch.cuda.synchronize()
    assert torch.equal(c[:m], y.clamp(min=0)) and bool((c[m:] == 7.0).all())
    # (about 2^30 ones: more than fp16 holds)
    assert float(sums[0]) == float("inf") and bool((sums[1:] == 7.0).all())


def test_the_longest_depth(gpu):
    """One row by one column of 2^31 - 1024 elements in K ranges; ones at both ends and at the borders of the ranges, so that the
    sum counts what was multiplied (and stays below 2^11, a whole number that fp16 holds)"""
    k = (1 << 31) - 1024
    a, b = (torch.zeros(k, device="cuda:0", dtype=torch.float16) for _ in range(2))
    places = {0, 1, 63, 64, k - 1, k - 2, k - 1024, 1 << 30, (1 << 30) - 1}
    for ranges in (31, 32):
        length = ((k + ranges - 1) // ranges + 63) // 64 * 64
        for r in range(1, ranges):
            places.update(range(r * length - 3, r * length + 3))
    index = torch.tensor(sorted(places), device="cuda:0")
    a[index], b[index] = 1.0, 1.0
    for split, turned in ((0, False), (31, True), (32, False)):
        api.override_parameters(0, "Xlayer", 16, {"TILE_VARIANT": 0, "SPLIT_K": split})
        try:
            c = torch.zeros(1, device="cuda:0", dtype=torch.float16)
            api.gemmEpilogue(None, 1, 1, k, a, b, c, 1 if turned else k, k if turned else 1, 1, a_transp=turned, b_transp=turned)
            torch.cuda.synchronize()
        finally:
            api.override_parameters(0, "Xlayer", 16, {"TILE_VARIANT": 0, "SPLIT_K": 0})
        assert float(c) == len(places), (split, float(c), len(places))


def test_lines_up_to_the_reach_of_32_bits(gpu):
    """17 rows of the longest that 16 rows may have (the sixteenth 4.3e9 bytes behind the first); ones where both operands have
    them count what was multiplied. A piece more is refused. Then features as many as eight depths reach."""
    m, k = 17, 143165552
    a, b = torch.zeros(m, k, device="cuda:0", dtype=torch.float16), torch.zeros(2, k, device="cuda:0", dtype=torch.float16)
    places = torch.tensor([0, 1, 31, 32, 12345678, k // 2, k - 33, k - 2, k - 1], device="cuda:0")
    b[0, places] = 1.0
    b[1, places[:4]] = 2.0
    for row in range(m):
        a[row, places[:1 + row % 9]] = 1.0 + row
    c = torch.zeros(m, 2, device="cuda:0", dtype=torch.float16)
    api.gemmEpilogue(None, m, 2, k, a, b, c, k, k, 2, b_transp=True)
    torch.cuda.synchronize()
    want = [[(1 + row) * (1 + row % 9), (1 + row) * 2 * min(4, 1 + row % 9)] for row in range(m)]
    assert c.tolist() == want
    long = torch.zeros(m * (k + 16), device="cuda:0", dtype=torch.float16)
    with pytest.raises(api.CLBlastError) as error:
        api.gemmEpilogue(None, m, 1, k + 16, long, long, c, k + 16, k + 16, 1, b_transp=True)
    assert error.value.status == -1017
    del a, b, long
    n, k = 306783328, 9
    g = torch.Generator(device="cuda:0").manual_seed(13)
    a = torch.tensor([[1.0, 2.0, -1.0, 3.0, -2.0, 1.0, 4.0, -3.0, 2.0]], device="cuda:0", dtype=torch.float16)
    b = torch.empty(k, n, device="cuda:0", dtype=torch.float16)
    want = torch.zeros(n, device="cuda:0")
    for row in range(k):
        b[row] = torch.randint(-8, 9, (n,), generator=g, device="cuda:0", dtype=torch.int8)
        want += b[row].float() * float(a[0, row])  # (whole numbers: exact)
    c = torch.full((n + 3,), 7.0, device="cuda:0", dtype=torch.float16)
    api.gemmEpilogue(None, 1, n, k, a, b, c, k, n, n)
    torch.cuda.synchronize()
    assert torch.equal(c[:n].float(), want) and bool((c[n:] == 7.0).all())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
def test_one_bias_for_all_groups(gpu, dtype):
    g = torch.Generator(device="cuda:0").manual_seed(14)
    m, n, k, groups = 150, 72, 40, 4
    a, b, bias = (torch.randn(*shape, generator=g, device="cuda:0").to(dtype) for shape in ((m, k), (groups, k, n), (n,)))
    bounds = [0, 30, 30, 101, 150]
    offsets = torch.tensor(bounds, device="cuda:0")
    c = torch.zeros(m, n, dtype=dtype, device="cuda:0")
    api.gemmGrouped(None, groups, m, n, k, a, b, c, offsets, k, n, n, k * n, bias=bias, bias_stride=0, activation="silu")
    torch.cuda.synchronize()
    for e in range(groups):
        rows = slice(bounds[e], bounds[e + 1])
        want, bound, _, _ = ref.epilogue(a[rows].double(), b[e].double(), dtype, 1.0, bias.double(), "silu")
        ref.check(c[rows], want, bound, "group %d" % e)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
def test_the_activations_input_as_the_result(gpu, dtype):
    """C of the activation's gradient in the place of Z, by two rows of a wavefront in flight and by rows side by side"""
    g = torch.Generator(device="cuda:0").manual_seed(15)
    for m, n in ((1, 1), (37, 9), (301, 520), (1030, 64)):
        y, z = (torch.randn(m, n, generator=g, device="cuda:0").to(dtype) for _ in range(2))
        want, bound, want_d, d_bound = ref.gradient(y.double(), torch.zeros(m, n, device="cuda:0", dtype=torch.float64), z.double(), "gelu", dtype)
        sums = torch.zeros(n, dtype=dtype, device="cuda:0")
        api.activationGradient(None, m, n, y, z, z, n, n, n, "gelu", bias_gradient=sums)
        torch.cuda.synchronize()
        ref.check(z, want, bound, "c of %d x %d" % (m, n))
        ref.check(sums, want_d, d_bound, "sums of %d x %d" % (m, n))


def test_the_most_groups(gpu):
    """65536 groups, most of one row, some of none or of more than a tile, found by offsets that begin inside their buffer"""
    g = torch.Generator(device="cuda:0").manual_seed(16)
    groups, n, k = 65536, 8, 16
    sizes = torch.ones(groups, dtype=torch.int64)
    sizes[5::7] = 0
    sizes[100], sizes[40000], sizes[65535] = 300, 65, 129
    ends = sizes.cumsum(0)
    m = int(ends[-1]) + 3
    offsets = torch.cat([torch.tensor([77, 0, 0]), ends]).to("cuda:0")  # (two values in front of the first)
    owner = torch.repeat_interleave(torch.arange(groups), sizes).to("cuda:0")
    a = torch.randint(-4, 5, (m, k), generator=g, device="cuda:0").half()
    b = torch.randint(-4, 5, (groups, k, n), generator=g, device="cuda:0").half()
    c = torch.full((m, n), 7.0, device="cuda:0", dtype=torch.float16)
    api.gemmGrouped(None, groups, m, n, k, a, b, c, offsets, k, n, n, k * n, group_offsets_offset=2)
    grad = torch.full((groups, k, n), 7.0, device="cuda:0", dtype=torch.float16)
    api.gemmGroupedGradient(None, groups, m, k, n, a, c, grad, offsets, k, n, n, k * n, alpha=0.0625, group_offsets_offset=2)
    sums = torch.full((groups, n), 7.0, device="cuda:0", dtype=torch.float16)
    api.activationGradient(None, m, n, c, None, None, n, 0, 0, bias_gradient=sums, group_count=groups, group_offsets=offsets, group_offsets_offset=2)
    torch.cuda.synchronize()
    used = m - 3
    want = (a[:used].float()[:, :, None] * b[owner].float()).sum(1)  # (whole numbers up to 256: exact)
    assert torch.equal(c[:used].float(), want) and bool((c[used:] == 7.0).all())
    want_sums = torch.zeros(groups, n, device="cuda:0").index_add_(0, owner, want)
    assert torch.equal(sums, want_sums.half())
    outer = a[:used].float()[:, :, None] * want[:, None, :] * 0.0625
    assert torch.equal(grad, torch.zeros(groups, k, n, device="cuda:0").index_add_(0, owner, outer).half())
