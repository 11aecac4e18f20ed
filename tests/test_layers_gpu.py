"""Products with bias, activation and residual in their epilogue, their backward pass and products grouped by expert, against
the same in 64 bits (tests/layer_reference.py, where the bounds are derived): types, transposes, odd sizes, leading dimensions
and offsets, every tile, K ranges, groups of every kind, what must not be read and what must not be written."""
import pytest
import torch

from clblast_amd import api
from tests import layer_reference as ref

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float16, torch.float32)
KINDS = ("none", "relu", "gelu", "gelu_tanh", "silu")
BITS = {torch.bfloat16: 16, torch.float16: 16, torch.float32: 32}


class Forced:
    """A tile (0: by rule) and a number of K ranges (0: by rule) for the layer products, while the block lasts"""

    def __init__(self, dtype, variant, split=0):
        self.bits, self.values = BITS[dtype], {"TILE_VARIANT": variant, "SPLIT_K": split}

    def __enter__(self):
        api.override_parameters(0, "Xlayer", self.bits, self.values)

    def __exit__(self, *_):
        api.override_parameters(0, "Xlayer", self.bits, {"TILE_VARIANT": 0, "SPLIT_K": 0})


def generator(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def place(values, dtype, ld, offset, fill=float("nan")):
    """A row-major matrix of leading dimension `ld` that starts `offset` elements into a buffer of `fill`: (buffer, view)"""
    rows, cols = values.shape
    buffer = torch.full((offset + rows * ld + 5,), fill, dtype=dtype, device="cuda:0")
    view = buffer[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(values)
    return buffer, view


def normal(g, rows, cols, scale=1.0):
    return torch.randn(rows, cols, generator=g, device="cuda:0") * scale


def untouched(buffer, before, view):
    """Everything of the buffer outside the view as it was, bit for bit"""
    now, was = buffer.clone(), before.clone()
    for t in (now, was):
        t.as_strided(view.shape, view.stride(), view.storage_offset()).zero_()
    kind = torch.int32 if buffer.dtype == torch.float32 else torch.int16
    assert torch.equal(now.view(kind), was.view(kind)), "elements outside the matrix were written"


def run_epilogue(dtype, m, n, k, a_transp=False, b_transp=False, kind="none", bias=True, pre=False, beta=0.0, alpha=1.0, pads=(0, 0, 0),
                 offsets=(0, 0, 0), seed=1, in_place=False):
    g = generator(seed)
    a_pad, b_pad, c_pad = pads
    a_shape, b_shape = ((k, m) if a_transp else (m, k)), ((n, k) if b_transp else (k, n))
    a_buffer, a = place(normal(g, *a_shape), dtype, a_shape[1] + a_pad, offsets[0])
    b_buffer, b = place(normal(g, *b_shape, k ** -0.5), dtype, b_shape[1] + b_pad, offsets[1])
    c_buffer, c = place(torch.full((m, n), float("nan"), device="cuda:0"), dtype, n + c_pad, offsets[2])
    bias_buffer, bias_view = place(normal(g, 1, n), dtype, n, offsets[2])
    r_buffer, r = place(normal(g, m, n), dtype, n + c_pad, offsets[0]) if beta != 0.0 else (None, None)
    z_buffer, z = place(torch.full((m, n), float("nan"), device="cuda:0"), dtype, n + b_pad, offsets[1]) if pre else (None, None)
    wide_a, wide_b = a.double(), b.double()
    want, bound, want_z, z_bound = ref.epilogue(
        wide_a.T if a_transp else wide_a, wide_b.T if b_transp else wide_b, dtype, alpha, bias_view[0].double() if bias else None, kind, beta,
        None if r is None else r.double())
    if in_place:
        c.copy_(r)
        r_buffer, r = c_buffer, c
    before = c_buffer.clone()
    z_before = None if z is None else z_buffer.clone()
    api.gemmEpilogue(None, m, n, k, a_buffer, b_buffer, c_buffer, a.stride(0), b.stride(0), c.stride(0), alpha=alpha, beta=beta,
                     a_transp=a_transp, b_transp=b_transp, bias=bias_buffer if bias else None, activation=kind, pre=z_buffer,
                     pre_ld=0 if z is None else z.stride(0), residual=r_buffer, residual_ld=0 if r is None else r.stride(0),
                     a_offset=a.storage_offset(), b_offset=b.storage_offset(), c_offset=c.storage_offset(),
                     bias_offset=bias_view.storage_offset(), pre_offset=0 if z is None else z.storage_offset(),
                     residual_offset=0 if r is None else r.storage_offset())
    torch.cuda.synchronize()
    ref.check(c, want, bound, "c")
    untouched(c_buffer, before, c)
    if pre:
        ref.check(z, want_z, z_bound, "pre")
        untouched(z_buffer, z_before, z)
    return c.clone()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_epilogue_small(gpu, dtype, kind):
    run_epilogue(dtype, 37, 72, 48, kind=kind, pre=True, beta=0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("a_transp", (False, True))
@pytest.mark.parametrize("b_transp", (False, True))
def test_epilogue_transposes_strides_and_offsets(gpu, dtype, a_transp, b_transp):
    """Aligned rows, then rows that start at every parity (16-bit operands are then copied first)"""
    run_epilogue(dtype, 130, 140, 100, a_transp, b_transp, "gelu", pre=True, beta=-1.5, alpha=0.75, pads=(4, 8, 2), offsets=(2, 4, 6))
    run_epilogue(dtype, 131, 139, 101, a_transp, b_transp, "silu", pre=True, beta=2.0, alpha=-1.25, pads=(0, 2, 0), offsets=(1, 3, 5), seed=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("variant", (1, 2, 3, 4, 5))
@pytest.mark.parametrize("split", (1, 3))
def test_epilogue_every_tile_and_k_ranges(gpu, dtype, variant, split):
    """Whole and ragged tiles; every number of slabs up to the ring's, with and without a tail"""
    if dtype == torch.float32 and variant == 2:
        pytest.skip("the 256 x 256 tile is for 16-bit data")
    with Forced(dtype, variant, split):
        run_epilogue(dtype, 256, 512, 128, False, True, "gelu", pre=True, beta=1.0)
        run_epilogue(dtype, 301, 266, 330, False, True, "none", beta=1.0, seed=3)
        run_epilogue(dtype, 301, 266, 330, True, False, "relu", seed=4)
        for k in (1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 97):
            run_epilogue(dtype, 40, 70, k, False, k % 2 == 0, "none", seed=k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", ((1, 1, 1), (1, 1, 700), (1, 1000, 1), (700, 1, 3), (1, 4096, 2048), (2, 64, 4096), (17, 1000, 1024), (33, 2050, 513)))
def test_epilogue_few_rows_or_features(gpu, dtype, m, n, k):
    run_epilogue(dtype, m, n, k, b_transp=True, kind="gelu_tanh", pre=True, beta=1.0)
    run_epilogue(dtype, m, n, k, kind="silu", bias=False, seed=5)


@pytest.mark.parametrize("dtype", TYPES)
def test_epilogue_residual_in_place_and_nothing_read_that_must_not_be(gpu, dtype):
    run_epilogue(dtype, 70, 90, 64, kind="gelu", beta=1.0, in_place=True)
    # (beta = 0: run_epilogue's C is NaN before the call, and the padding of every operand is)
    run_epilogue(dtype, 70, 91, 65, kind="gelu", beta=0.0, pads=(3, 5, 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_epilogue_large(gpu, dtype):
    run_epilogue(dtype, 1030, 2056, 1032, b_transp=True, kind="gelu", pre=True, beta=1.0)


def run_gradient(dtype, m, n, k, a_transp=False, b_transp=False, kind="gelu", alpha=1.0, pad=0, offset=0, seed=1, sums=True):
    g = generator(seed)
    a_shape, b_shape = ((k, m) if a_transp else (m, k)), ((n, k) if b_transp else (k, n))
    a_buffer, a = place(normal(g, *a_shape), dtype, a_shape[1] + pad, offset)
    b_buffer, b = place(normal(g, *b_shape, k ** -0.5), dtype, b_shape[1] + pad, offset)
    z_buffer, z = place(normal(g, m, n, 2.0), dtype, n + pad, offset)
    c_buffer, c = place(torch.full((m, n), float("nan"), device="cuda:0"), dtype, n + pad, offset)
    d_buffer, d = place(torch.full((1, n), float("nan"), device="cuda:0"), dtype, n, offset)
    wide_a, wide_b = a.double().T if a_transp else a.double(), b.double().T if b_transp else b.double()
    y = alpha * (wide_a @ wide_b)
    y_error = (k + 8) * 2.0 ** -24 * abs(alpha) * (wide_a.abs() @ wide_b.abs())
    want, bound, want_d, d_bound = ref.gradient(y, y_error, z.double(), kind, dtype)
    before, d_before = c_buffer.clone(), d_buffer.clone()
    api.gemmActivationGradient(None, m, n, k, a_buffer, b_buffer, z_buffer if kind != "none" else None, c_buffer, a.stride(0), b.stride(0),
                               z.stride(0), c.stride(0), alpha=alpha, a_transp=a_transp, b_transp=b_transp, activation=kind,
                               bias_gradient=d_buffer if sums else None, a_offset=offset, b_offset=offset, pre_offset=offset, c_offset=offset,
                               bias_gradient_offset=offset)
    torch.cuda.synchronize()
    ref.check(c, want, bound, "c")
    untouched(c_buffer, before, c)
    if sums:
        ref.check(d, want_d[None], d_bound[None], "bias_gradient")
        untouched(d_buffer, d_before, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_gradient_small(gpu, dtype, kind):
    run_gradient(dtype, 70, 72, 48, kind=kind)
    run_gradient(dtype, 71, 73, 49, kind=kind, pad=2, offset=3, alpha=-0.5, sums=kind != "relu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("variant", (1, 2, 3, 4, 5))
@pytest.mark.parametrize("split", (1, 4))
def test_gradient_every_tile_and_k_ranges(gpu, dtype, variant, split):
    if dtype == torch.float32 and variant == 2:
        pytest.skip("the 256 x 256 tile is for 16-bit data")
    with Forced(dtype, variant, split):
        run_gradient(dtype, 515, 300, 260, b_transp=True)
        run_gradient(dtype, 256, 256, 256, a_transp=True, kind="silu", seed=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", ((1, 1, 1), (1, 1000, 64), (2000, 3, 17), (1000, 1032, 520), (8, 512, 4096)))
def test_gradient_sizes(gpu, dtype, m, n, k):
    run_gradient(dtype, m, n, k, kind="gelu_tanh")


def offsets_of(sizes, first=0):
    ends = [first]
    for size in sizes:
        ends.append(ends[-1] + size)
    return torch.tensor(ends, dtype=torch.int64, device="cuda:0")


GROUPINGS = {
    "one": (0, [50], 0), "even": (0, [32, 32, 32, 32], 0), "empty ones": (0, [0, 40, 0, 0, 7, 0], 0), "all empty": (5, [0, 0, 0], 9),
    "rows of nobody": (11, [20, 1, 33], 17), "single rows": (0, [1] * 70, 3), "one large": (0, [3, 400, 2], 1),
    "many": (2, [(i * 7) % 5 for i in range(200)], 4),
}


def run_activation(dtype, rows, n, kind, grouping=None, pad=0, offset=0, seed=1, result=True, sums=True, in_place=False):
    g = generator(seed)
    first, sizes = (0, [rows]) if grouping is None else grouping
    y_buffer, y = place(normal(g, rows, n), dtype, n + pad, offset)
    z_buffer, z = place(normal(g, rows, n, 2.0), dtype, n + pad, offset)
    last = first + sum(sizes)
    for t in (y, z):  # rows of nobody are not read
        t[:first] = float("nan")
        t[last:] = float("nan")
    c_buffer, c = (y_buffer, y) if in_place else place(torch.full((rows, n), 7.0, device="cuda:0"), dtype, n + pad, offset)
    d_buffer, d = place(torch.full((len(sizes), n), float("nan"), device="cuda:0"), dtype, n, offset)
    wide_y, wide_z = y.double(), z.double()
    before = c_buffer.clone()
    api.activationGradient(None, rows, n, y_buffer, z_buffer if kind != "none" else None, c_buffer if result else None, n + pad, n + pad, n + pad,
                           activation=kind, bias_gradient=d_buffer if sums else None, group_count=len(sizes),
                           group_offsets=None if grouping is None else offsets_of(sizes, first), y_offset=offset, pre_offset=offset,
                           c_offset=offset, bias_gradient_offset=offset)
    torch.cuda.synchronize()
    at = first
    for index, size in enumerate(sizes):
        want, bound, want_d, d_bound = ref.gradient(wide_y[at:at + size], torch.zeros_like(wide_y[at:at + size]), wide_z[at:at + size], kind, dtype)
        if result:
            ref.check(c[at:at + size], want, bound, "c of group %d" % index)
        if sums:
            ref.check(d[index], want_d, d_bound, "bias_gradient of group %d" % index)
        at += size
    untouched(c_buffer, before, c[first:last] if result else c[:0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_activation_gradient(gpu, dtype, kind):
    run_activation(dtype, 70, 72, kind)
    run_activation(dtype, 71, 73, kind, pad=2, offset=3)
    run_activation(dtype, 300, 520, kind, result=False)
    run_activation(dtype, 33, 9, kind, sums=False)
    run_activation(dtype, 33, 1, kind, in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grouping", sorted(GROUPINGS))
def test_activation_gradient_by_group(gpu, dtype, grouping):
    first, sizes, after = GROUPINGS[grouping]
    run_activation(dtype, first + sum(sizes) + after, 136, "silu", (first, sizes))
    run_activation(dtype, first + sum(sizes) + after, 131, "gelu", (first, sizes), in_place=True)


def run_grouped(dtype, sizes, n, k, first=0, after=0, b_transp=False, kind="none", bias=True, pre=False, beta=0.0, alpha=1.0, pad=0, offset=0,
                shared=False, seed=1):
    g = generator(seed)
    m, groups = first + sum(sizes) + after, len(sizes)
    last = m - after
    a_buffer, a = place(normal(g, m, k), dtype, k + pad, offset)
    a[:first] = float("nan")
    a[last:] = float("nan")
    shape = (n, k) if b_transp else (k, n)
    count = 1 if shared else groups
    b_ld = shape[1] + pad
    b_buffer, b = place(normal(g, count * shape[0], shape[1], k ** -0.5), dtype, b_ld, offset)
    b_stride = 0 if shared else shape[0] * b_ld
    bias_buffer, bias_view = place(normal(g, groups, n), dtype, n + pad, offset)
    c_buffer, c = place(normal(g, m, n) if beta else torch.full((m, n), float("nan"), device="cuda:0"), dtype, n + pad, offset)
    z_buffer, z = place(torch.full((m, n), 3.0, device="cuda:0"), dtype, n + pad, offset) if pre else (None, None)
    old = c.double()
    before, z_before = c_buffer.clone(), None if z is None else z_buffer.clone()
    api.gemmGrouped(None, groups, m, n, k, a_buffer, b_buffer, c_buffer, offsets_of(sizes, first), a.stride(0), b_ld, c.stride(0), b_stride,
                    alpha=alpha, beta=beta, b_transp=b_transp, bias=bias_buffer if bias else None, bias_stride=n + pad, activation=kind,
                    pre=z_buffer, pre_ld=0 if z is None else z.stride(0), a_offset=offset, b_offset=offset, c_offset=offset,
                    bias_offset=offset, pre_offset=offset)
    torch.cuda.synchronize()
    at = first
    for index, size in enumerate(sizes):
        rows = slice(at, at + size)
        at += size
        here = 0 if shared else index
        w = b[here * shape[0]:(here + 1) * shape[0]].double()
        want, bound, want_z, z_bound = ref.epilogue(a[rows].double(), w.T if b_transp else w, dtype, alpha,
                                                    bias_view[index].double() if bias else None, kind, beta, old[rows])
        ref.check(c[rows], want, bound, "c of group %d" % index)
        if pre:
            ref.check(z[rows], want_z, z_bound, "pre of group %d" % index)
    untouched(c_buffer, before, c[first:last])
    if pre:
        untouched(z_buffer, z_before, z[first:last])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grouping", sorted(GROUPINGS))
@pytest.mark.parametrize("b_transp", (False, True))
def test_grouped(gpu, dtype, grouping, b_transp):
    first, sizes, after = GROUPINGS[grouping]
    run_grouped(dtype, sizes, 136, 72, first, after, b_transp, "silu", pre=True)
    run_grouped(dtype, sizes, 67, 33, first, after, b_transp, "none", beta=0.5, alpha=-1.5, pad=2, offset=1, seed=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("variant", (1, 2, 3, 4, 5))
def test_grouped_every_tile(gpu, dtype, variant):
    if dtype == torch.float32 and variant == 2:
        pytest.skip("the 256 x 256 tile is for 16-bit data")
    with Forced(dtype, variant, 5):  # (K ranges are for products without groups: none here)
        run_grouped(dtype, [300, 0, 17, 256, 1], 520, 200, 0, 3, True, "gelu", pre=True)
        run_grouped(dtype, [31, 64, 300], 600, 96, 7, 0, False, "none", beta=1.0)
        run_grouped_gradient(dtype, [300, 0, 17, 256, 1], 300, 520)


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_with_one_matrix_for_all(gpu, dtype):
    run_grouped(dtype, [5, 0, 70], 80, 64, shared=True, b_transp=True)
    run_grouped(dtype, [5, 0, 70], 81, 63, shared=True)


def run_grouped_gradient(dtype, sizes, m, n, first=0, after=0, beta=0.0, alpha=1.0, pad=0, offset=0, seed=1):
    g = generator(seed)
    k, groups = first + sum(sizes) + after, len(sizes)
    last = k - after
    a_buffer, a = place(normal(g, k, m), dtype, m + pad, offset)
    b_buffer, b = place(normal(g, k, n), dtype, n + pad, offset)
    for t in (a, b):
        t[:first] = float("nan")
        t[last:] = float("nan")
    c_ld = n + pad
    c_buffer, c = place(normal(g, groups * m, n) if beta else torch.full((groups * m, n), float("nan"), device="cuda:0"), dtype, c_ld, offset)
    old = c.double()
    before = c_buffer.clone()
    api.gemmGroupedGradient(None, groups, k, m, n, a_buffer, b_buffer, c_buffer, offsets_of(sizes, first), m + pad, n + pad, c_ld, m * c_ld,
                            alpha=alpha, beta=beta, a_offset=offset, b_offset=offset, c_offset=offset)
    torch.cuda.synchronize()
    at = first
    for index, size in enumerate(sizes):
        rows, mine = slice(at, at + size), slice(index * m, (index + 1) * m)
        at += size
        want, bound, _, _ = ref.epilogue(a[rows].double().T, b[rows].double(), dtype, alpha, None, "none", beta, old[mine])
        ref.check(c[mine], want, bound, "c of group %d" % index)
    untouched(c_buffer, before, c)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("grouping", sorted(GROUPINGS))
def test_grouped_gradient(gpu, dtype, grouping):
    first, sizes, after = GROUPINGS[grouping]
    run_grouped_gradient(dtype, sizes, 72, 136, first, after)
    run_grouped_gradient(dtype, sizes, 33, 67, first, after, beta=-0.5, alpha=2.0, pad=2, offset=1, seed=2)


def test_offsets_that_lead_outside_are_clamped(gpu):
    """Nothing outside the matrices is read or written whatever the offsets say; groups that are in order still hold"""
    dtype, m, n, k = torch.bfloat16, 40, 72, 64
    g = generator(3)
    a, b = normal(g, m, k).to(dtype), normal(g, 4 * n, k, k ** -0.5).to(dtype)
    c = torch.full((m + 8, n), 5.0, dtype=dtype, device="cuda:0")
    offsets = torch.tensor([-(1 << 40), 10, 25, 1 << 40, 1 << 50], dtype=torch.int64, device="cuda:0")
    api.gemmGrouped(None, 4, m, n, k, a, b, c, offsets, k, k, n, n * k, b_transp=True)
    torch.cuda.synchronize()
    for index, (begin, end) in enumerate(((0, 10), (10, 25), (25, 40))):
        want, bound, _, _ = ref.epilogue(a[begin:end].double(), b[index * n:(index + 1) * n].double().T, dtype)
        ref.check(c[begin:end], want, bound, "group %d" % index)
    assert bool((c[m:] == 5.0).all())
    for values in ([40, 30, 20, 10, 0], [0, 40, 0, 40, 0], [7, 7, 7, 7, 7]):
        offsets = torch.tensor(values, dtype=torch.int64, device="cuda:0")
        api.gemmGrouped(None, 4, m, n, k, a, b, c, offsets, k, k, n, n * k, b_transp=True)
        sums = torch.zeros(5, n, dtype=dtype, device="cuda:0")
        api.activationGradient(None, m, n, c, c, None, n, n, 0, "gelu", bias_gradient=sums, group_count=4, group_offsets=offsets)
        result = torch.zeros(4, k, n, dtype=dtype, device="cuda:0")
        api.gemmGroupedGradient(None, 4, m, k, n, a, c, result, offsets, k, n, n, k * n)
        torch.cuda.synchronize()
        assert bool((c[m:] == 5.0).all()) and bool((sums[4] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("split", (1, 3))
def test_two_teams_along_the_depth(gpu, dtype, split):
    """The tile whose depth two sets of wavefronts share: every parity of slabs, depths that leave the second set a part of a
    slab or nothing, all transposes, sums in the bias gradient, groups"""
    with Forced(dtype, 6, split):
        for k in (1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 80, 95, 96, 97, 127, 128, 129, 160, 191, 192, 193, 320, 321, 1000):
            for a_transp in (False, True):
                for b_transp in (False, True):
                    run_epilogue(dtype, 70, 66, k, a_transp, b_transp, "none", beta=1.0, seed=k)
        run_epilogue(dtype, 256, 512, 128, False, True, "gelu", pre=True, beta=1.0)
        run_epilogue(dtype, 301, 266, 330, False, True, "silu", pre=True, beta=1.0, in_place=True, seed=3)
        run_gradient(dtype, 515, 300, 260, b_transp=True)
        run_gradient(dtype, 256, 256, 256, a_transp=True, kind="silu", seed=2)
        run_grouped(dtype, [300, 0, 17, 256, 1], 520, 200, 0, 3, True, "gelu", pre=True)
        run_grouped(dtype, [31, 64, 300], 600, 96, 7, 0, False, "none", beta=1.0)
        run_grouped_gradient(dtype, [300, 0, 17, 256, 1, 32, 33], 300, 520)
        run_grouped_gradient(dtype, [300, 0, 17, 256, 1, 32, 33], 65, 66, 3, 5, beta=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_teams_read_nothing_beyond_the_depth(gpu, dtype):
    """NaN behind every line of both operands, at depths that end inside a slab, at its end and before the second team's part"""
    g = generator(60)
    m, n = 70, 66
    with Forced(dtype, 6, 1):
        for k in (1, 7, 16, 33, 48, 64, 65, 97, 130):
            for a_transp in (False, True):
                for b_transp in (False, True):
                    a_buffer, a = place(normal(g, *((k, m) if a_transp else (m, k))), dtype, (m if a_transp else k) + 66, 2)
                    b_buffer, b = place(normal(g, *((n, k) if b_transp else (k, n))), dtype, (k if b_transp else n) + 66, 2)
                    for buffer, view in ((a_buffer, a), (b_buffer, b)):
                        values = view.clone()
                        buffer.fill_(float("nan"))
                        view.copy_(values)
                    c = torch.zeros(m, n, dtype=dtype, device="cuda:0")
                    api.gemmEpilogue(None, m, n, k, a_buffer, b_buffer, c, a.stride(0), b.stride(0), n, a_transp=a_transp, b_transp=b_transp,
                                     a_offset=a.storage_offset(), b_offset=b.storage_offset())
                    torch.cuda.synchronize()
                    wide_a, wide_b = a.double(), b.double()
                    want, bound, _, _ = ref.epilogue(wide_a.T if a_transp else wide_a, wide_b.T if b_transp else wide_b, dtype)
                    ref.check(c, want, bound, "k = %d" % k)
