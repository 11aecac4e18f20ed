"""The layer products as they are used: a feed-forward block and a block of experts trained through them, against automatic
differentiation in 64 bits; recorded into a graph and replayed; on other streams than the current one; with offsets and strides
beyond 32 bits; the same call again with the same bits."""
import threading

import pytest
import torch

import clblast_amd
from clblast_amd import api
from tests import layer_reference as ref

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float16, torch.float32)
# A chain of products in the storage type: every tensor in between is rounded (half a step, 2^-8, 2^-11 or 2^-24 of a value),
# and an error that enters a product of k random terms leaves it with the same size relative to the result's root mean
# square. Four roundings at most lie between the inputs and a gradient here, and activations enlarge one by at most 1.13:
# 4 * 1.13^2 * 2^-8 = 0.02 of the root mean square for a typical element; the bound is on the relative Frobenius norm, where
# rounding errors are uniform in +- half a step (a factor of sqrt(1/3)): below 4 * 1.13^2 / sqrt(3) = 3 half steps.
NORM = {torch.bfloat16: 3 * 2.0 ** -8, torch.float16: 3 * 2.0 ** -11, torch.float32: 3 * 2.0 ** -20}


def generator(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def near(got, want, dtype, what):
    error = float((got.double() - want).norm() / want.norm())
    assert error <= NORM[dtype], (what, error)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ("gelu", "silu"))
def test_training_step_of_a_feed_forward_block(gpu, dtype, kind):
    """Y = X + act(X W1 + b1) W2^T + b2 and all of its gradients"""
    g = generator(1)
    tokens, width, hidden = 333, 264, 520
    draw = lambda scale, *shape: (torch.randn(*shape, generator=g, device="cuda:0") * scale).to(dtype)
    x, w1, b1 = draw(1, tokens, width), draw(width ** -0.5, width, hidden), draw(0.1, hidden)
    w2, b2, dy = draw(hidden ** -0.5, width, hidden), draw(0.1, width), draw(1, tokens, width)
    z, h, y = (torch.empty(tokens, n, dtype=dtype, device="cuda:0") for n in (hidden, hidden, width))
    api.gemmEpilogue(None, tokens, hidden, width, x, w1, h, width, hidden, hidden, bias=b1, activation=kind, pre=z, pre_ld=hidden)
    api.gemmEpilogue(None, tokens, width, hidden, h, w2, y, hidden, hidden, width, b_transp=True, bias=b2, beta=1.0, residual=x, residual_ld=width)
    dz, db1, db2 = torch.empty_like(z), torch.empty_like(b1), torch.empty_like(b2)
    dw1, dw2, dx = torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(x)
    api.activationGradient(None, tokens, width, dy, None, None, width, 0, 0, bias_gradient=db2)
    api.gemmEpilogue(None, width, hidden, tokens, dy, h, dw2, width, hidden, hidden, a_transp=True)
    api.gemmActivationGradient(None, tokens, hidden, width, dy, w2, z, dz, width, hidden, hidden, hidden, activation=kind, bias_gradient=db1)
    api.gemmEpilogue(None, width, hidden, tokens, x, dz, dw1, width, hidden, hidden, a_transp=True)
    api.gemmEpilogue(None, tokens, width, hidden, dz, w1, dx, hidden, hidden, width, b_transp=True, beta=1.0, residual=dy, residual_ld=width)
    torch.cuda.synchronize()
    leaves = [t.double().requires_grad_() for t in (x, w1, b1, w2, b2)]
    X, W1, B1, W2, B2 = leaves
    Y = X + ref.act(X @ W1 + B1, kind) @ W2.T + B2
    Y.backward(dy.double())
    near(y, Y.detach(), dtype, "y")
    for name, got, leaf in zip(("dx", "dw1", "db1", "dw2", "db2"), (dx, dw1, db1, dw2, db2), leaves):
        near(got, leaf.grad, dtype, name)


@pytest.mark.parametrize("dtype", TYPES)
def test_training_step_of_a_block_of_experts(gpu, dtype):
    """Y_g = silu(X_g W1_g + b1_g) W2_g^T for ragged groups, one of them empty, rows of nobody at the end, and its gradients"""
    g = generator(2)
    sizes, width, hidden = [40, 0, 131, 1, 77], 136, 200
    groups, used, rows = len(sizes), sum(sizes), sum(sizes) + 7
    offsets = torch.tensor([0] + sizes, device="cuda:0").cumsum(0)
    draw = lambda scale, *shape: (torch.randn(*shape, generator=g, device="cuda:0") * scale).to(dtype)
    x, w1, b1 = draw(1, rows, width), draw(width ** -0.5, groups, width, hidden), draw(0.1, groups, hidden)
    w2, dy = draw(hidden ** -0.5, groups, width, hidden), draw(1, rows, width)
    z, h, dh, dz = (torch.full((rows, hidden), 9.0, dtype=dtype, device="cuda:0") for _ in range(4))
    y, dx = (torch.full((rows, width), 9.0, dtype=dtype, device="cuda:0") for _ in range(2))
    dw1, dw2, db1 = torch.empty_like(w1), torch.empty_like(w2), torch.empty_like(b1)
    each = width * hidden
    api.gemmGrouped(None, groups, rows, hidden, width, x, w1, h, offsets, width, hidden, hidden, each, bias=b1, activation="silu", pre=z, pre_ld=hidden)
    api.gemmGrouped(None, groups, rows, width, hidden, h, w2, y, offsets, hidden, hidden, width, each, b_transp=True)
    api.gemmGroupedGradient(None, groups, rows, width, hidden, dy, h, dw2, offsets, width, hidden, hidden, each)
    api.gemmGrouped(None, groups, rows, hidden, width, dy, w2, dh, offsets, width, hidden, hidden, each)
    api.activationGradient(None, rows, hidden, dh, z, dz, hidden, hidden, hidden, activation="silu", bias_gradient=db1, group_count=groups, group_offsets=offsets)
    api.gemmGroupedGradient(None, groups, rows, width, hidden, x, dz, dw1, offsets, width, hidden, hidden, each)
    api.gemmGrouped(None, groups, rows, width, hidden, dz, w1, dx, offsets, hidden, hidden, width, each, b_transp=True)
    torch.cuda.synchronize()
    leaves = [t.double().requires_grad_() for t in (x, w1, b1, w2)]
    X, W1, B1, W2 = leaves
    at, parts = 0, []
    for e, size in enumerate(sizes):
        parts.append(ref.act(X[at:at + size] @ W1[e] + B1[e], "silu") @ W2[e].T)
        at += size
    Y = torch.cat(parts)
    Y.backward(dy[:used].double())
    near(y[:used], Y.detach(), dtype, "y")
    near(dx[:used], X.grad[:used], dtype, "dx")
    for name, got, leaf in zip(("dw1", "db1", "dw2"), (dw1, db1, dw2), (W1, B1, W2)):
        near(got, leaf.grad, dtype, name)
        assert bool((got[1] == 0).all()), "the empty expert's " + name
    for t in (z, h, dh, dz, y, dx):
        assert bool((t[used:] == 9.0).all()), "rows of nobody"


def test_a_gradient_against_differences(gpu):
    """The step's own directional derivative in fp32. The loss is a sum of 96 * 80 products of order one: its two values are off
    by about sqrt(7680) * 2^-22 = 2e-5 (a few roundings of 2^-24 each), over 2h = 0.02 that is 1e-3; the third derivative adds
    h^2 / 6 times a sum of 7680 terms of order one and of either sign, 1.7e-5 * 88 * 2 = 3e-3. The bound is twelve times
    their sum; the derivative itself is of the order of sqrt(7680) = 88."""
    g = generator(3)
    m, n, k, h = 96, 80, 64, 0.01
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda:0")
    x, w, b, direction, weight = draw(m, k), draw(k, n) * k ** -0.5, draw(n), draw(k, n) * k ** -0.5, draw(m, n)

    def loss(matrix):
        y = torch.empty(m, n, device="cuda:0")
        api.gemmEpilogue(None, m, n, k, x, matrix.contiguous(), y, k, n, n, bias=b, activation="gelu")
        return float((y.double() * weight.double()).sum())

    z, dz, dw = torch.empty(m, n, device="cuda:0"), torch.empty(m, n, device="cuda:0"), torch.empty(k, n, device="cuda:0")
    y = torch.empty(m, n, device="cuda:0")
    api.gemmEpilogue(None, m, n, k, x, w, y, k, n, n, bias=b, activation="gelu", pre=z, pre_ld=n)
    api.activationGradient(None, m, n, weight, z, dz, n, n, n, activation="gelu")
    api.gemmEpilogue(None, k, n, m, x, dz, dw, k, n, n, a_transp=True)
    slope = float((dw.double() * direction.double()).sum())
    difference = (loss(w + h * direction) - loss(w - h * direction)) / (2 * h)
    assert abs(slope - difference) <= 0.05, (slope, difference)


def everything(t, stream=None):
    """Calls of all five operators, with K ranges, copies of unaligned operands and sums in the workspace"""
    m, n, k = 130, 264, 2048
    api.gemmEpilogue(stream, m, n, k, t["a"], t["b"], t["c"], k, k, n, b_transp=True, bias=t["bias"], activation="gelu", pre=t["z"], pre_ld=n)
    api.gemmEpilogue(stream, m, 71, 131, t["a"], t["b"], t["odd"], 131, 71, 71, activation="relu", a_offset=1, b_offset=3)
    api.gemmActivationGradient(stream, m, n, k, t["a"], t["b"], t["z"], t["dz"], k, k, n, n, b_transp=True, activation="gelu", bias_gradient=t["db"])
    api.activationGradient(stream, m, n, t["c"], t["z"], t["dz2"], n, n, n, activation="silu", bias_gradient=t["db2"], group_count=4, group_offsets=t["offsets"])
    api.gemmGrouped(stream, 4, m, 64, n, t["c"], t["b"], t["y"], t["offsets"], n, 64, 64, n * 64, activation="silu")
    api.gemmGroupedGradient(stream, 4, m, n, 64, t["c"], t["y"], t["dw"], t["offsets"], n, 64, 64, n * 64)


OUTPUTS = ("c", "z", "odd", "dz", "db", "dz2", "db2", "y", "dw")


def tensors(dtype, seed):
    g = generator(seed)
    m, n, k = 130, 264, 2048
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda:0").to(dtype)
    t = {"a": draw(m * k + 8), "b": draw(n * k + 8), "bias": draw(n), "offsets": torch.tensor([0, 30, 30, 99, 125], device="cuda:0")}
    for name, shape in zip(OUTPUTS, ((m, n), (m, n), (m, 71), (m, n), (n,), (m, n), (4, n), (m, 64), (4, n, 64))):
        t[name] = torch.zeros(shape, dtype=dtype, device="cuda:0")
    return t


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_call_gives_the_same_bits(gpu, dtype):
    first, second = tensors(dtype, 4), tensors(dtype, 4)
    for _ in range(3):
        everything(first)
        everything(second)
        torch.cuda.synchronize()
        for name in OUTPUTS:
            assert torch.equal(first[name], second[name]), name


@pytest.mark.parametrize("dtype", TYPES)
def test_recorded_into_a_graph(gpu, dtype):
    """Replays with other inputs and other groups against eager calls, with the program's own work in between"""
    t, other = tensors(dtype, 5), tensors(dtype, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(t)  # un-captured: the stream's scratch buffer now exists
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        everything(t)
    torch.cuda.synchronize()
    for replay, offsets in enumerate(([0, 30, 30, 99, 125], [0, 0, 0, 0, 130], [5, 6, 70, 71, 71], [0, 130, 130, 130, 130])):
        fresh = tensors(dtype, 10 + replay)
        for both in (t, other):
            for name in ("a", "b", "bias"):
                both[name].copy_(fresh[name])
            both["offsets"].copy_(torch.tensor(offsets, device="cuda:0"))
            for name in OUTPUTS:
                both[name].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        everything(other)
        torch.cuda.synchronize()
        for name in OUTPUTS:
            assert torch.equal(t[name], other[name]), (replay, name)
    assert clblast_amd.clear_cache() == 0


def test_streams_and_threads(gpu):
    """Four threads on streams of their own, two of them with the stream as an argument, against the same calls made alone"""
    wanted = {}
    for seed in range(4):
        t = tensors(torch.bfloat16, 20 + seed)
        everything(t)
        torch.cuda.synchronize()
        wanted[seed] = {name: t[name].clone() for name in OUTPUTS}
    failures = []

    def work(seed):
        try:
            stream = torch.cuda.Stream()
            t = tensors(torch.bfloat16, 20 + seed)
            torch.cuda.synchronize()
            for _ in range(5):
                if seed % 2:
                    everything(t, stream)
                else:
                    with torch.cuda.stream(stream):
                        everything(t)
            stream.synchronize()
            for name in OUTPUTS:
                if not torch.equal(t[name], wanted[seed][name]):
                    failures.append((seed, name))
        except Exception as error:  # noqa: BLE001 - reported by the main thread
            failures.append((seed, error))

    threads = [threading.Thread(target=work, args=(seed,)) for seed in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


def test_offsets_and_strides_beyond_32_bits(gpu):
    """Rows of C, of Z and of the residual 2^31 elements apart, an operand with lines further apart than the tiled kernel
    reaches, experts more than 2^32 bytes apart"""
    dtype, m, n, k = torch.bfloat16, 3, 72, 64
    g = generator(6)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda:0").to(dtype)
    far = (1 << 31) + 10
    big = torch.zeros(2 * far + n + 8, dtype=dtype, device="cuda:0")  # 8.6 GB
    a, b = draw(m, k), draw(n, k)
    residual = draw(m, n)
    rows = big.as_strided((m, n), (far, 1))
    rows.copy_(residual)
    want, bound, want_z, z_bound = ref.epilogue(a.double(), b.double().T, dtype, 1.0, None, "gelu", 1.0, residual.double())
    z = torch.zeros(m, n, dtype=dtype, device="cuda:0")
    api.gemmEpilogue(None, m, n, k, a, b, big, k, k, far, b_transp=True, activation="gelu", pre=z, pre_ld=n, beta=1.0, residual=big, residual_ld=far)
    torch.cuda.synchronize()
    ref.check(rows, want, bound, "rows of C far apart")
    ref.check(z, want_z, z_bound, "z")
    assert float(big[n:n + 4096].abs().max()) == 0.0 and float(big[far - 4096:far].abs().max()) == 0.0
    lines = (1 << 21) + 5
    rows_of_a = big[:].as_strided((m, k), (lines, 1))
    rows_of_a.copy_(a)
    c = torch.zeros(m, n, dtype=dtype, device="cuda:0")
    api.gemmEpilogue(None, m, n, k, big, b, c, lines, k, n, b_transp=True, activation="gelu")
    want, bound, _, _ = ref.epilogue(a.double(), b.double().T, dtype, kind="gelu")
    torch.cuda.synchronize()
    ref.check(c, want, bound, "lines of A far apart")
    experts = big.as_strided((2, n, k), (far, k, 1))
    weights = draw(2, n, k)
    experts.copy_(weights)
    offsets = torch.tensor([0, 1, 3], device="cuda:0")
    api.gemmGrouped(None, 2, m, n, k, a, big, c, offsets, k, k, n, far, b_transp=True)
    torch.cuda.synchronize()
    for e, (begin, end) in enumerate(((0, 1), (1, 3))):
        want, bound, _, _ = ref.epilogue(a[begin:end].double(), weights[e].double().T, dtype)
        ref.check(c[begin:end], want, bound, "expert %d" % e)
    result = big.as_strided((2, k, n), (far, n, 1))
    api.gemmGroupedGradient(None, 2, m, k, n, a, c, big, offsets, k, n, n, far)
    torch.cuda.synchronize()
    for e, (begin, end) in enumerate(((0, 1), (1, 3))):
        want, bound, _, _ = ref.epilogue(a[begin:end].double().T, c[begin:end].double(), dtype)
        ref.check(result[e], want, bound, "gradient of expert %d" % e)


def test_special_values(gpu):
    """Infinities and NaN stay in their rows and columns; a residual with beta = 0, rows of nobody and padding bring none in
    (the other tests fill those with NaN); large finite inputs of the activations give finite slopes"""
    for dtype in TYPES:
        g = generator(7)
        m, n, k = 70, 72, 40
        a, b = torch.randn(m, k, generator=g, device="cuda:0").to(dtype), torch.randn(k, n, generator=g, device="cuda:0").to(dtype)
        a[3, 5], a[9, 0] = float("nan"), float("inf")
        c = torch.zeros(m, n, dtype=dtype, device="cuda:0")
        api.gemmEpilogue(None, m, n, k, a, b, c, k, n, n)
        torch.cuda.synchronize()
        assert bool(c[3].isnan().all()) and bool((~c[9].isfinite()).all())
        rest = torch.ones(m, dtype=torch.bool, device="cuda:0")
        rest[3] = rest[9] = False
        assert bool(c[rest].isfinite().all())
        largest = torch.finfo(dtype).max
        z = torch.tensor([[-largest, largest, -200.0, 200.0, -1e4, 1e4, 0.0, -0.0]], device="cuda:0").to(dtype)
        one = torch.ones_like(z)
        for kind, ends in (("relu", (0, 1)), ("gelu", (0, 1)), ("gelu_tanh", (0, 1)), ("silu", (0, 1)), ("none", (1, 1))):
            out = torch.zeros_like(z)
            api.activationGradient(None, 1, 8, one, z, out, 8, 8, 8, activation=kind)
            torch.cuda.synchronize()
            expected = [ends[0], ends[1]] * 3
            assert [float(v) for v in out[0, :6]] == expected, (dtype, kind, out)


def test_python_calls_on_other_devices_and_types(gpu):
    a = torch.zeros(8, 8, dtype=torch.float64, device="cuda:0")
    with pytest.raises(ValueError, match="data-type"):
        api.gemmEpilogue(None, 8, 8, 8, a, a, a, 8, 8, 8)
    a = a.half()
    with pytest.raises(ValueError, match="one GPU"):
        api.gemmEpilogue(None, 8, 8, 8, a, a.cpu(), a, 8, 8, 8)
    offsets = torch.tensor([0, 8], dtype=torch.int32, device="cuda:0")
    with pytest.raises(ValueError, match="64-bit"):
        api.gemmGrouped(None, 1, 8, 8, 8, a, a, a, offsets, 8, 8, 8, 64)
    with pytest.raises(clblast_amd.CLBlastError) as error:
        api.gemmGrouped(None, 0, 8, 8, 8, a, a, a, offsets.long(), 8, 8, 8, 64)
    assert error.value.status == -2049
    with pytest.raises(clblast_amd.CLBlastError) as error:
        api.gemmEpilogue(None, 8, 8, 8, a, a, a, 7, 8, 8)
    assert error.value.status == -1016


@pytest.mark.parametrize("dtype", TYPES)
def test_lines_of_an_operand_beyond_the_tiled_kernels_reach(gpu, dtype):
    """Either operand with lines 2^23 and more elements apart, as it is and transposed"""
    g = generator(30)
    m, n, k = 37, 72, 24
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda:0").to(dtype)
    for ld in ((1 << 23) - 2, 1 << 23, (1 << 23) + 6):
        big = torch.full((37 * ld + 64,), float("nan"), dtype=dtype, device="cuda:0")
        for transposed in (False, True):
            a, b = draw(m, k), draw(k, n)
            want, bound, _, _ = ref.epilogue(a.double(), b.double(), dtype)
            far = big.as_strided((k, m) if transposed else (m, k), (ld, 1))
            far.copy_(a.T if transposed else a)
            c = torch.zeros(m, n, dtype=dtype, device="cuda:0")
            api.gemmEpilogue(None, m, n, k, big, b, c, ld, n, n, a_transp=transposed)
            torch.cuda.synchronize()
            ref.check(c, want, bound, "a, %d apart" % ld)
            # the other operand: its first 37 columns (rows) alone, so that the same memory does
            far = big.as_strided((37, k) if transposed else (k, 37), (ld, 1))
            far.copy_(b[:, :37].T if transposed else b[:, :37])
            c = torch.zeros(m, 37, dtype=dtype, device="cuda:0")
            api.gemmEpilogue(None, m, 37, k, a, big, c, k, ld, 37, b_transp=transposed)
            torch.cuda.synchronize()
            ref.check(c, want[:, :37], bound[:, :37], "b, %d apart" % ld)


def test_sums_of_many_overlapping_groups(gpu):
    """Offsets that go back and forth make every other group as long as the whole matrix: together the groups have far more
    chunks of rows than there are (2^31 and more). What the sums hold then is not specified; nothing around them is touched, and
    groups in order give the right sums right behind such a call."""
    rows, groups = 1 << 25, 1 << 14
    y = torch.ones(rows, 1, dtype=torch.float16, device="cuda:0")
    sums = torch.full((groups + 128,), 7.0, dtype=torch.float16, device="cuda:0")
    offsets = torch.zeros(groups + 1, dtype=torch.int64, device="cuda:0")
    offsets[1::2] = rows
    api.activationGradient(None, rows, 1, y, None, None, 1, 0, 0, bias_gradient=sums, group_count=groups, group_offsets=offsets, bias_gradient_offset=64)
    torch.cuda.synchronize()
    assert bool((sums[:64] == 7.0).all()) and bool((sums[groups + 64:] == 7.0).all())
    offsets = torch.arange(groups + 1, device="cuda:0") * (rows // groups)
    api.activationGradient(None, rows, 1, y, None, None, 1, 0, 0, bias_gradient=sums, group_count=groups, group_offsets=offsets, bias_gradient_offset=64)
    torch.cuda.synchronize()
    assert bool((sums[64:groups + 64] == rows // groups).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_results_of_groups_side_by_side(gpu, dtype):
    """The groups' results as columns of one matrix, in place"""
    g = generator(31)
    sizes, m, n = [9, 0, 70], 40, 72
    k, groups = sum(sizes), len(sizes)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda:0").to(dtype)
    a, b, c = draw(k, m), draw(k, n), draw(m, groups * n + 5)
    old = c.clone()
    offsets = torch.tensor([0] + sizes, device="cuda:0").cumsum(0)
    api.gemmGroupedGradient(None, groups, k, m, n, a, b, c, offsets, m, n, groups * n + 5, n, beta=1.0)
    torch.cuda.synchronize()
    at = 0
    for e, size in enumerate(sizes):
        columns = slice(e * n, (e + 1) * n)
        want, bound, _, _ = ref.epilogue(a[at:at + size].double().T, b[at:at + size].double(), dtype, 1.0, None, "none", 1.0, old[:, columns].double())
        ref.check(c[:, columns], want, bound, "group %d" % e)
        at += size
    assert torch.equal(c[:, groups * n:], old[:, groups * n:])


def test_two_graphs_of_one_stream(gpu):
    """Two graphs captured on a stream share its scratch: replayed on it in turn, with eager calls in between"""
    dtype = torch.bfloat16
    first, second, other = (tensors(dtype, seed) for seed in (40, 41, 42))
    wanted = []
    for seed in (40, 41, 42):
        t = tensors(dtype, seed)
        everything(t)
        torch.cuda.synchronize()
        wanted.append({name: t[name].clone() for name in OUTPUTS})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(other)
    side.synchronize()
    graphs = []
    for t in (first, second):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            everything(t)
    torch.cuda.synchronize()
    for _ in range(3):
        for t in (first, second, other):
            for name in OUTPUTS:
                t[name].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
            everything(other)
        side.synchronize()
        for t, want in zip((first, second, other), wanted):
            for name in OUTPUTS:
                assert torch.equal(t[name], want[name]), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", (1, 3, 8, 20, 129, 256, 300))
def test_narrow_matrices_and_long_sums(gpu, dtype, n):
    """Rows that take less than a wavefront side by side, with and without groups, whole and at odd places, against 64 bits. A
    sum of p products of normal numbers in any order of fp32: p roundings of 2^-24 of a partial sum at most, which stays
    below sum |.|, then its own rounding."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    g = generator(50 + n)
    m = 5003
    y, z = (torch.randn(m, n + 2, generator=g, device="cuda:0").to(dtype) for _ in range(2))
    c = torch.full((m, n + 2), 9.0, dtype=dtype, device="cuda:0")
    bounds = [0, 0, 1, 700, 703, 703, 4990]
    offsets = torch.tensor(bounds, device="cuda:0")
    want = torch.where(z > 0, y, torch.zeros_like(y))  # relu: nothing is rounded
    for groups in (None, offsets):
        count = 1 if groups is None else len(bounds) - 1
        ranges = [(0, m)] if groups is None else list(zip(bounds[:-1], bounds[1:]))
        c.fill_(9.0)
        sums = torch.full((count * n + 2,), 9.0, dtype=dtype, device="cuda:0")
        api.activationGradient(None, m, n, y, z, c, n + 2, n + 2, n + 2, "relu", bias_gradient=sums, group_count=count, group_offsets=groups,
                               y_offset=1, pre_offset=1, c_offset=1, bias_gradient_offset=1)
        torch.cuda.synchronize()
        assert torch.equal(c[:ranges[-1][1], 1:-1], want[:ranges[-1][1], 1:-1])
        assert bool((c[:, 0] == 9.0).all()) and bool((c[:, -1] == 9.0).all()) and bool((c[ranges[-1][1]:] == 9.0).all())
        assert float(sums[0]) == 9.0 and float(sums[-1]) == 9.0
        for e, (begin, end) in enumerate(ranges):
            part = want[begin:end, 1:-1].double()
            exact, size = part.sum(0), part.abs().sum(0)
            error = (sums[1 + e * n:1 + (e + 1) * n].double() - exact).abs()
            bound = size * (end - begin) * 2.0 ** -24 * (1 + half) + exact.abs() * half + 2.0 ** -25
            assert bool((error <= bound).all()), (e, float((error - bound).max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_activations_at_the_infinities(gpu, dtype):
    """The limits of the functions and of their slopes; a NaN stays one"""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[-inf, inf, nan, 0.0, -inf, inf, nan, 0.0]], device="cuda:0").to(dtype)
    for kind, left, right in (("relu", 0.0, inf), ("gelu", 0.0, inf), ("gelu_tanh", 0.0, inf), ("silu", 0.0, inf), ("none", -inf, inf)):
        for rows in (1, 300):  # an edge, and whole tiles
            ones = torch.ones(rows, 1, device="cuda:0").to(dtype)
            wide = z.repeat(1, 64).contiguous()
            n = wide.shape[1]
            c = torch.zeros(rows, n, dtype=dtype, device="cuda:0")
            api.gemmEpilogue(None, rows, n, 1, ones, wide, c, 1, n, n, activation=kind)
            torch.cuda.synchronize()
            assert bool((c[:, 0::4] == left).all()) and bool((c[:, 1::4] == right).all()) and bool(c[:, 2::4].isnan().all()) and bool((c[:, 3::4] == 0).all()), kind
        out = torch.zeros_like(z)
        api.activationGradient(None, 1, 8, torch.ones_like(z), z, out, 8, 8, 8, activation=kind)
        torch.cuda.synchronize()
        assert float(out[0, 0]) == (1.0 if kind == "none" else 0.0) and float(out[0, 1]) == 1.0, (kind, out)
        assert bool(out[0, 2].isnan()) or kind in ("relu", "none"), (kind, out)
